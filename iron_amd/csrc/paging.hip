// Pages of a KV cache: appending rows to sequences, forking and copying
// sequences, packing the pool and giving pages back.
//
// State, all of it in device memory, so that a serving loop needs no host
// round trip for it and can be captured whole:
//   k_pages, v_pages  (layers, num_pages, n_kv_heads, page_size, head_dim)
//   page_table        (num_seqs, max_pages) int32: position t of sequence s is
//                     row t % page_size of page page_table[s][t / page_size];
//                     an entry outside [0, num_pages) is a hole (no page)
//   seq_lens          (num_seqs) int32
//   page_refs         (num_pages) int32: how many table entries hold the page; 0 = free
// Pages are given out lowest number first, in the order of the requests, so
// every result is a function of the inputs alone (no free list whose order
// would depend on atomics). What a request needs is decided by one workgroup
// (a prefix sum over the requests and a search for that many zeros in
// page_refs); the data then moves in a launch that fills the chip.
#include "iron_common.hpp"
#include "int4_rows.hpp"
#include "../../include/iron_hip.h"

#include <algorithm>
#include <climits>

namespace iron {
namespace {

constexpr int kPlan = 1024;         // threads of the one workgroup that plans a call
constexpr int kMaxSeqs = 8192;
constexpr int kMaxRequests = 8192;  // sequences of an append, pairs of a fork: what is known of them lives in LDS
constexpr int kMaxRows = 1 << 20;   // of one append: the prefix sums stay in 32 bits whatever row_starts holds

// What became of a request (enum iron_page_status).
constexpr int PAGE_DONE = IRON_PAGE_DONE, PAGE_INVALID = IRON_PAGE_INVALID, PAGE_NO_ROOM = IRON_PAGE_NO_ROOM,
              PAGE_NOT_OWN = IRON_PAGE_NOT_OWN;

struct Pool {
  unsigned char* k;
  unsigned char* v;
  int* table;
  int* lens;
  int* refs;
  int num_layers, num_pages, page_size, num_seqs, max_pages;
  int n_kv_heads;
  int row_chunks;  // 16-byte chunks of one head's row
  __device__ __forceinline__ bool in_pool(int page) const {
    return static_cast<unsigned>(page) < static_cast<unsigned>(num_pages);
  }
  __device__ __forceinline__ int pages_of(int len) const { return (len + page_size - 1) / page_size; }
  __device__ __forceinline__ bool len_fits(long long len) const {
    return len >= 0 && len <= static_cast<long long>(max_pages) * page_size;
  }
  __device__ __forceinline__ long long page_chunks() const {
    return static_cast<long long>(n_kv_heads) * page_size * row_chunks;
  }
};

// Exclusive prefix sum over the workgroup's NT threads; total to every thread.
// tmp: NT / 64 values of LDS. Every thread calls it.
template <int NT, typename T>
__device__ __forceinline__ T block_scan(T x, T* tmp, T& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  T incl = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const T y = __shfl_up(incl, d, 64);
    if (lane >= d) incl += y;
  }
  __syncthreads();  // tmp is free: every thread has left an earlier call
  if (lane == 63) tmp[w] = incl;
  __syncthreads();
  T base = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    const T y = tmp[i];
    base += i < w ? y : 0;
    sum += y;
  }
  total = sum;
  return base + incl - x;
}

// need[0..n) -> its exclusive prefix sum in place (LDS); returns the sum.
__device__ int scan_requests(int* need, int n, int* tmp) {
  int carry = 0;
  for (int b = 0; b < n; b += kPlan) {
    const int i = b + threadIdx.x;
    const int x = i < n ? need[i] : 0;
    int total;
    const int e = block_scan<kPlan>(x, tmp, total);
    if (i < n) need[i] = carry + e;
    carry += total;
  }
  __syncthreads();
  return carry;
}

// Bit j: the count of page base + j is 0 (and there is such a page).
__device__ __forceinline__ unsigned free4(const int4& r, int base, int num_pages) {
  const unsigned zeros = static_cast<unsigned>(r.x == 0) | static_cast<unsigned>(r.y == 0) << 1 |
                         static_cast<unsigned>(r.z == 0) << 2 | static_cast<unsigned>(r.w == 0) << 3;
  const int left = num_pages - base;
  return zeros & (left >= 4 ? 15u : (1u << max(left, 0)) - 1);
}

// The counts of pages base .. base + 3 (base a multiple of 4), and of those that there are.
__device__ __forceinline__ int4 counts4(const int* refs, int base, int num_pages) {
  if (base + 4 <= num_pages) return *reinterpret_cast<const int4*>(refs + base);
  int4 r = make_int4(0, 0, 0, 0);
  if (base < num_pages) r.x = refs[base];
  if (base + 1 < num_pages) r.y = refs[base + 1];
  if (base + 2 < num_pages) r.z = refs[base + 2];
  return r;
}

// The lowest `want` free pages into list (global), as many as there are;
// returns how many were found (at most want). `first` is counts4 of pages
// 4 tid .. + 3, which the caller asks for before all else: most calls need no
// more than those. Then four such reads of each thread at a time, as far as needed.
__device__ int find_free(const int* refs, int num_pages, int want, int* list, int* tmp, const int4& first) {
  constexpr int kAhead = 4;
  int found = 0;
  int4 r[kAhead] = {first};
  for (int b = 0, n = 1; b < num_pages && found < want; b += 4 * kPlan * n, n = kAhead) {
    if (b) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) r[k] = counts4(refs, b + 4 * (k * kPlan + static_cast<int>(threadIdx.x)), num_pages);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (k >= n || found >= want) break;
      const int p0 = b + 4 * (k * kPlan + static_cast<int>(threadIdx.x));
      unsigned zeros = free4(r[k], p0, num_pages);
      int total;
      int at = found + block_scan<kPlan>(static_cast<int>(__popc(zeros)), tmp, total);
      while (zeros && at < want) {
        list[at++] = p0 + __ffs(zeros) - 1;
        zeros &= zeros - 1;
      }
      found += total;
    }
  }
  __syncthreads();
  return min(found, want);
}

// Index of the request that gets granted page r: the last one whose exclusive
// prefix is <= r (requests that need none have the next one's prefix).
__device__ __forceinline__ int request_of(const int* first, int n, int r) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= r)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Request i got its pages: its last one is among the `have` that were found. A
// request that the pages run out for gets none of them, and no later one that
// needs some does: what is granted stays a prefix of the list.
__device__ __forceinline__ bool granted(const int* first, int i, int n, int want, int have) {
  const int end = i + 1 < n ? first[i + 1] : want;
  return end == first[i] || end <= have;
}

// ------------------------------------------------------------------ append ----
struct AppendArgs {
  Pool pool;
  const uint4* k_new;  // (layers, num_nodes, n_kv_heads, row_chunks)
  const uint4* v_new;
  const int* rows;        // (num_rows) source rows
  const int* row_starts;  // (num_seqs + 1)
  int* status;            // (num_seqs)
  int* begin;             // workspace (num_seqs): the length before the call, or -1 where nothing is appended
  int* list;              // workspace (list_cap): pages given out
  int num_nodes, num_rows, list_cap;
};

// Rows [first, stop) of the call are sequence s's, all of them or none: a range
// that leaves the rows or ends before its start is no range (one without rows is,
// wherever it lies).
__device__ __forceinline__ bool range_fits(const AppendArgs& a, int first, int stop) {
  return first == stop || (0 <= first && first < stop && stop <= a.num_rows);
}

// row_starts decreases somewhere: a range with rows that starts below an earlier
// entry would take rows that an earlier range has, so its sequence gets none. The
// largest entry so far is a running maximum over the workgroup. Every thread calls it.
__device__ void refuse_overlaps(const AppendArgs& a, int* need, int* grow, int* tmp) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n = a.pool.num_seqs;
  int carry = INT_MIN;
  for (int b = 0; b < n; b += kPlan) {
    const int s = b + threadIdx.x, x = s < n ? a.row_starts[s] : INT_MIN;
    int top = x;
    for (int d = 1; d < 64; d *= 2) {
      const int y = __shfl_up(top, d, 64);
      if (lane >= d) top = max(top, y);
    }
    __syncthreads();  // tmp is free
    if (lane == 63) tmp[w] = top;
    __syncthreads();
    top = max(top, carry);
    for (int i = 0; i < kPlan / 64; ++i) {
      if (i < w) top = max(top, tmp[i]);
      carry = max(carry, tmp[i]);
    }
    if (s < n && grow[s] >> 2 > 0 && x < top) {
      need[s] = 0;
      grow[s] = PAGE_INVALID;
    }
  }
}

// Decides which sequences grow, gives them pages and moves their lengths. One
// workgroup, bound by its chain of dependent reads: the counts that the search
// for free pages begins with are asked for first, and what was read of the
// sequences stays in LDS (8 sequences 4.0 -> 2.7 us, four prompts 6.4 -> 4.5).
// Judging row_starts costs 0.2 us: whether it decreases anywhere goes through LDS
// behind the barrier that was there.
__global__ __launch_bounds__(kPlan) void append_plan_kernel(AppendArgs a) {
  __shared__ int need[kMaxRequests];
  __shared__ int lens[kMaxRequests];
  __shared__ int grow[kMaxRequests];  // rows to append and, in the lowest two bits, the status
  __shared__ int tmp[kPlan / 64];
  static_assert(kMaxRows <= 1 << 28 && PAGE_NOT_OWN < 4, "both fit");
  const Pool& p = a.pool;
  const int4 front = counts4(p.refs, 4 * threadIdx.x, p.num_pages);
  bool decreases = false;
  for (int s = threadIdx.x; s < p.num_seqs; s += kPlan) {
    const int first = a.row_starts[s], stop = a.row_starts[s + 1], len = p.lens[s];
    const bool fits = range_fits(a, first, stop);
    const int count = fits ? stop - first : 0;
    int st = PAGE_DONE, n = 0;
    decreases |= stop < first;
    if (!fits || !p.len_fits(len)) {
      st = PAGE_INVALID;
    } else if (!p.len_fits(static_cast<long long>(len) + count)) {
      st = PAGE_NO_ROOM;
    } else if (count > 0) {
      if (len % p.page_size) {  // the first rows go to the sequence's last page: it has to be there, and its alone
        const int page = p.table[static_cast<long long>(s) * p.max_pages + len / p.page_size];
        if (!p.in_pool(page) || p.refs[page] != 1) st = PAGE_NOT_OWN;
      }
      if (st == PAGE_DONE) n = p.pages_of(len + count) - p.pages_of(len);
    }
    need[s] = n;
    lens[s] = len;
    grow[s] = count << 2 | st;
  }
  decreases = __ballot(decreases) != 0;
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = decreases;
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int i = 0; i < kPlan / 64; ++i) any |= tmp[i];
  if (__builtin_expect(any, 0)) refuse_overlaps(a, need, grow, tmp);
  const int want = scan_requests(need, p.num_seqs, tmp);
  const int have = find_free(p.refs, p.num_pages, min(want, a.list_cap), a.list, tmp, front);
  for (int s = threadIdx.x; s < p.num_seqs; s += kPlan) {
    int st = grow[s] & 3;
    if (st == PAGE_DONE && !granted(need, s, p.num_seqs, want, have)) st = PAGE_NO_ROOM;
    a.status[s] = st;
    a.begin[s] = st == PAGE_DONE ? lens[s] : -1;
    if (st == PAGE_DONE) p.lens[s] = lens[s] + (grow[s] >> 2);
  }
  for (int r = threadIdx.x; r < have; r += kPlan) {
    const int s = request_of(need, p.num_seqs, r);
    if (!granted(need, s, p.num_seqs, want, have)) continue;
    const int page = a.list[r];
    p.refs[page] = 1;
    p.table[static_cast<long long>(s) * p.max_pages + p.pages_of(lens[s]) + (r - need[s])] = page;
  }
}

// One row of the call in `group` layers: K and V of every KV head. Bound by
// memory: 437 MB (four prompts, 16 layers) in 91 us, 4.8 TB/s.
__global__ __launch_bounds__(256) void append_rows_kernel(AppendArgs a, int group) {
  __shared__ int owner, to_pos;
  const Pool& p = a.pool;
  const int r = blockIdx.x, src = a.rows[r];
  if (threadIdx.x == 0) owner = -1;
  __syncthreads();
  for (int s = threadIdx.x; s < p.num_seqs; s += 256) {
    const int first = a.row_starts[s], stop = a.row_starts[s + 1], begin = a.begin[s];  // one round trip
    if (first <= r && r < stop && begin >= 0) {  // one sequence at most: the plan lets no two share a row
      owner = s;
      to_pos = begin + (r - first);
    }
  }
  __syncthreads();
  const int s = owner, pos = to_pos;
  if (s < 0) return;
  const int page = p.table[static_cast<long long>(s) * p.max_pages + pos / p.page_size];
  if (!p.in_pool(page)) return;
  const bool real = static_cast<unsigned>(src) < static_cast<unsigned>(a.num_nodes);
  const unsigned per_row = p.n_kv_heads * p.row_chunks;  // chunks of a layer's K (or V) row
  const int l0 = blockIdx.y * group, layers = min(group, p.num_layers - l0);
  const long long to_row = static_cast<long long>(pos % p.page_size) * p.row_chunks;
  for (unsigned t = threadIdx.x; t < layers * 2 * per_row; t += 256) {
    const unsigned lk = t / per_row, c = t - lk * per_row;
    const unsigned h = c / p.row_chunks, e = c - h * p.row_chunks;
    const long long l = l0 + (lk >> 1);
    const uint4* from = lk & 1 ? a.v_new : a.k_new;
    uint4* to = reinterpret_cast<uint4*>(lk & 1 ? p.v : p.k);
    uint4 x = make_uint4(0, 0, 0, 0);
    if (real) x = from[(l * a.num_nodes + src) * per_row + c];
    to[(l * p.num_pages + page) * p.page_chunks() + static_cast<long long>(h) * p.page_size * p.row_chunks + to_row + e] = x;
  }
}

// ------------------------------------------------------- 4-bit rows ----
// Where 16 rows of a call go or come from: the owner of each (the first sequence
// whose range holds it, -1 for none), its page and its row there. Every thread
// calls it; `begin_of(s, begin)` gives the position of the first row of s's range
// and whether s counts, `end_of(s)` the positions that s has.
constexpr int kTile = 16;

struct RowPlace {
  int owner[kTile];
  int page[kTile];  // -1: none
  int at[kTile];
};

template <typename F, typename E>
__device__ __forceinline__ void place_rows(const Pool& p, const int* row_starts, int num_rows, int r0, RowPlace& place, F begin_of, E end_of) {
  const int tid = threadIdx.x;
  if (tid < kTile) place.owner[tid] = INT_MAX;
  __syncthreads();
  for (int s = tid; s < p.num_seqs; s += 256) {
    const int first = row_starts[s], stop = row_starts[s + 1];
    int begin;
    if (begin_of(s, begin))
      for (int r = max(first, r0); r < min(stop, r0 + kTile); ++r) atomicMin(place.owner + (r - r0), s);
  }
  __syncthreads();
  if (tid < kTile) {
    int s = place.owner[tid], page = -1, at = 0, begin;
    if (s == INT_MAX || r0 + tid >= num_rows) s = -1;
    if (s >= 0 && begin_of(s, begin)) {
      const long long pos = begin + (static_cast<long long>(r0 + tid) - row_starts[s]);
      if (pos >= 0 && pos < end_of(s) && pos < static_cast<long long>(p.max_pages) * p.page_size) {
        page = p.table[static_cast<long long>(s) * p.max_pages + pos / p.page_size];
        at = static_cast<int>(pos % p.page_size);
      }
    }
    place.owner[tid] = s;
    place.page[tid] = p.in_pool(page) ? page : -1;
    place.at[tid] = at;
  }
  __syncthreads();
}

template <bool F16>
__device__ __forceinline__ float wide16(unsigned x) {
  if constexpr (F16) return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(x)));
  return __uint_as_float(x << 16);
}

// 16 rows of the call, `items` of the (layer, K or V, head) planes to a workgroup: a
// wave takes a plane, a lane eight values of a row at a time, so that both sides are
// read and written in whole lines. The lanes of a quarter (2, or 4 with head_dim 128)
// find its range together. 6,670 rows (301 MB) in 83 us, 3.6 TB/s: 44 us of it are
// the quantizing's instructions, and a wave's loads ahead of them saved nothing.
template <int D, bool F16>
__global__ __launch_bounds__(256) void append4_rows_kernel(AppendArgs a, int items) {
  constexpr int kRow = kInt4Row<D>, L = D / 8, kTurns = kTile * L / 64;  // lanes of a row, rows of a lane
  __shared__ RowPlace place;
  const Pool& p = a.pool;
  const int r0 = blockIdx.x * kTile, lane = threadIdx.x & 63, e = lane % L;
  place_rows(p, a.row_starts, a.num_rows, r0, place, [&](int s, int& begin) { return (begin = a.begin[s]) >= 0; }, [](int) { return INT_MAX; });
  const int H = p.n_kv_heads, planes = p.num_layers * 2 * H, stop = min(planes, (static_cast<int>(blockIdx.y) + 1) * items);
  int page[kTurns], at[kTurns], src[kTurns];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int r = i * (64 / L) + lane / L;
    page[i] = place.owner[r] < 0 ? -1 : place.page[r];
    at[i] = place.at[r];
    src[i] = a.rows[min(r0 + r, a.num_rows - 1)];
  }
  for (int x = blockIdx.y * items + (threadIdx.x >> 6); x < stop; x += 4) {
    const int lk = x / H, h = x - lk * H, l = lk >> 1;
    uint4 y[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const bool real = static_cast<unsigned>(src[i]) < static_cast<unsigned>(a.num_nodes);
      y[i] = make_uint4(0, 0, 0, 0);
      if (real) y[i] = (lk & 1 ? a.v_new : a.k_new)[((static_cast<long long>(l) * a.num_nodes + src[i]) * H + h) * L + e];
    }
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const unsigned w[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
      float v[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = wide16<F16>(w[j] & 0xffffu);
        v[2 * j + 1] = wide16<F16>(w[j] >> 16);
      }
      unsigned codes;
      const unsigned pair = int4_quantize<L / 4>(v, codes);
      if (page[i] < 0) continue;
      unsigned char* to = (lk & 1 ? p.v : p.k) + (((static_cast<long long>(l) * p.num_pages + page[i]) * H + h) * p.page_size + at[i]) * kRow;
      *reinterpret_cast<unsigned*>(to + e * 4) = codes;
      if (e % (L / 4) == 0) *reinterpret_cast<unsigned*>(to + D / 2 + e / (L / 4) * 4) = pair;
    }
  }
}

struct GatherArgs {
  Pool pool;
  const int* begins;      // (num_seqs)
  const int* row_starts;  // (num_seqs + 1)
  uint4* k_out;           // (layers, num_rows, n_kv_heads, D / 8)
  uint4* v_out;
  int num_rows;
};

// The other way round: 16 rows of the result. Bound by memory (1.72 GB in 340 us, 5.0 TB/s).
template <int D, bool F16>
__global__ __launch_bounds__(256) void gather4_rows_kernel(GatherArgs a, int items) {
  constexpr int kRow = kInt4Row<D>, L = D / 8, kTurns = kTile * L / 64;
  __shared__ RowPlace place;
  const Pool& p = a.pool;
  const int r0 = blockIdx.x * kTile, lane = threadIdx.x & 63, e = lane % L;
  place_rows(p, a.row_starts, a.num_rows, r0, place, [&](int s, int& begin) { return begin = a.begins[s], true; }, [&](int s) { return p.lens[s]; });
  const int H = p.n_kv_heads, planes = p.num_layers * 2 * H, stop = min(planes, (static_cast<int>(blockIdx.y) + 1) * items);
  int page[kTurns], at[kTurns];
  bool mine[kTurns];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int r = i * (64 / L) + lane / L;
    mine[i] = place.owner[r] >= 0;
    page[i] = place.page[r];
    at[i] = place.at[r];
  }
  for (int x = blockIdx.y * items + (threadIdx.x >> 6); x < stop; x += 4) {
    const int lk = x / H, h = x - lk * H, l = lk >> 1;
    unsigned codes[kTurns], pair[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      codes[i] = pair[i] = 0;
      if (page[i] >= 0) {
        const unsigned char* from = (lk & 1 ? p.v : p.k) + (((static_cast<long long>(l) * p.num_pages + page[i]) * H + h) * p.page_size + at[i]) * kRow;
        codes[i] = *reinterpret_cast<const unsigned*>(from + e * 4);
        pair[i] = *reinterpret_cast<const unsigned*>(from + D / 2 + e / (L / 4) * 4);
      }
    }
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      unsigned y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float lo = int4_dequant(pair[i], int4_code(codes[i], 2 * j)), hi = int4_dequant(pair[i], int4_code(codes[i], 2 * j + 1));
        if constexpr (F16)
          y[j] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(lo)) | static_cast<unsigned>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(hi))) << 16;
        else
          y[j] = cvt_pk_bf16(lo, hi);
      }
      const int r = r0 + i * (64 / L) + lane / L;
      if (mine[i]) (lk & 1 ? a.v_out : a.k_out)[((static_cast<long long>(l) * a.num_rows + r) * H + h) * L + e] = make_uint4(y[0], y[1], y[2], y[3]);
    }
  }
}

// Planes to a workgroup: as many as leave 4096 workgroups, in fours, one to a wave
// (6,670 rows of 16 layers and 8 heads of 64, appended and read back: 4096 workgroups
// 157 us, 2048 171, 8192 156, 16384 184).
int planes_of(int num_rows, int planes) {
  const long long all = static_cast<long long>((num_rows + kTile - 1) / kTile) * planes;
  const long long least = std::max<long long>(4, (planes + 32767) / 32768);  // the grid's second dimension ends at 65535
  return static_cast<int>(std::max(least, std::min<long long>(planes, all / 4096 / 4 * 4)));
}

// ----------------------------------------------------------- page copies ----
// Pages to copy: the first rows[i] rows (rows null: all) of every head of page
// src[i] to page dst[i], K and V, all layers. No page is both a source and a
// destination. One workgroup copies a page of a layer's K or V, 4 KiB at a time,
// each waited for. With thousands of pages that is bound by memory (pages of 16
// positions: four whole sequences, 557 MB, in 111 us, and a third of a pool packed,
// 917 MB, in 183 us: 5.0 TB/s); with few and large ones by its round trips (whole
// calls, 8 heads of 128: one fork's last page of 255 of 256 rows, one layer, 28 us
// for 2 MB, of 1023 of 1024 rows 96 us for 8 MB, 168 us with 16 layers, 134 MB;
// 12 us at pages of 16).
struct Copies {
  const int* src;
  const int* dst;
  const int* rows;
  const int* count;
};

__device__ __forceinline__ void copy_pages(const Pool& p, const Copies& c, int block, int blocks) {
  const long long tasks = static_cast<long long>(*c.count) * p.num_layers * 2;
  const long long size = p.page_chunks();
  for (long long t = block; t < tasks; t += blocks) {
    const int i = static_cast<int>(t / (2 * p.num_layers)), lk = static_cast<int>(t - static_cast<long long>(i) * 2 * p.num_layers);
    uint4* base = reinterpret_cast<uint4*>(lk & 1 ? p.v : p.k) + static_cast<long long>(lk >> 1) * p.num_pages * size;
    const uint4* from = base + c.src[i] * size;
    uint4* to = base + c.dst[i] * size;
    const int rows = c.rows ? c.rows[i] : p.page_size;
    if (rows == p.page_size) {
      for (long long x = threadIdx.x; x < size; x += 256) to[x] = from[x];
    } else {
      const unsigned part = rows * p.row_chunks, stride = p.page_size * p.row_chunks;
      for (unsigned x = threadIdx.x; x < part * p.n_kv_heads; x += 256) {
        const unsigned h = x / part, at = h * stride + (x - h * part);
        to[at] = from[at];
      }
    }
  }
}

// -------------------------------------------------------------------- fork ----
struct ForkArgs {
  Pool pool;
  const int* forks;  // (num_forks, 2): parent, child
  int* status;       // (num_forks)
  int* len;          // workspace (num_forks): the parent's length, or -1 where nothing is done
  int* first;        // workspace (num_forks): where the pair's pages begin in dst
  int* dst;          // workspace (list_cap): pages given out,
  int* src;          //   the pages copied to them
  int* rows;         //   and how many rows of each
  int* count;        // workspace: copies to make
  int num_forks, list_cap, share;
};

// One workgroup: which pairs count (each child's first, found in LDS), their
// pages, and the copies to make. Bound by its chain of dependent reads: 16 pairs
// 4.4 us (5.8 with the claims in global memory and no counts asked for early),
// four whole copies 8.4.
__global__ __launch_bounds__(kPlan) void fork_plan_kernel(ForkArgs a) {
  __shared__ int need[kMaxRequests];
  __shared__ int claim[kMaxSeqs];  // the first pair that names the child
  __shared__ int tmp[kPlan / 64];
  __shared__ int copies;
  const Pool& p = a.pool;
  const int ps = p.page_size, n = a.num_forks;
  const int4 front = counts4(p.refs, 4 * threadIdx.x, p.num_pages);
  if (threadIdx.x == 0) copies = 0;
  auto slot = [&](int s) { return static_cast<unsigned>(s) < static_cast<unsigned>(p.num_seqs); };
  auto row = [&](int s) { return p.table + static_cast<long long>(s) * p.max_pages; };
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int child = a.forks[2 * i + 1];
    if (slot(child)) claim[child] = n;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int child = a.forks[2 * i + 1];
    if (slot(child)) atomicMin(claim + child, i);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int parent = a.forks[2 * i], child = a.forks[2 * i + 1];
    int st = PAGE_INVALID, len = -1, pages = 0;
    if (slot(parent) && slot(child) && parent != child && claim[child] == i) {
      const int to = p.lens[child], from = p.lens[parent];
      if (to == 0 && p.len_fits(from)) {
        st = PAGE_DONE;
        len = from;
        pages = a.share ? (len % ps != 0 && p.in_pool(row(parent)[len / ps])) : 0;
      }
    }
    a.status[i] = st;
    a.len[i] = len;
    need[i] = pages;
  }
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (!a.share) {  // a page for every page that the parent has
    for (int i = wave; i < n; i += kPlan / 64) {
      const int pages = a.len[i] < 0 ? 0 : p.pages_of(a.len[i]);
      const int* from = row(a.forks[2 * i]);
      int found = 0;
      for (int e = lane; e < pages; e += 64) found += p.in_pool(from[e]);
      for (int d = 32; d; d >>= 1) found += __shfl_xor(found, d, 64);
      if (lane == 0) need[i] = found;
    }
    __syncthreads();
  }
  const int want = scan_requests(need, n, tmp);
  const int have = find_free(p.refs, p.num_pages, min(want, a.list_cap), a.dst, tmp, front);
  for (int i = threadIdx.x; i < n; i += kPlan) {
    if (a.len[i] < 0) continue;
    if (!granted(need, i, n, want, have)) {
      a.status[i] = PAGE_NO_ROOM;
      a.len[i] = -1;
      continue;
    }
    p.lens[a.forks[2 * i + 1]] = a.len[i];
    a.first[i] = need[i];
    const int end = i + 1 < n ? need[i + 1] : want;
    if (end > need[i]) atomicMax(&copies, end);
  }
  __syncthreads();
  if (threadIdx.x == 0) *a.count = copies;
  for (int r = threadIdx.x; r < copies; r += kPlan) p.refs[a.dst[r]] = 1;
  if (a.share) {
    for (int r = threadIdx.x; r < copies; r += kPlan) {
      const int i = request_of(need, n, r), len = a.len[i];
      a.src[r] = row(a.forks[2 * i])[len / ps];
      a.rows[r] = len % ps;
    }
    return;
  }
  for (int i = wave; i < n; i += kPlan / 64) {
    const int len = a.len[i];
    if (len < 0) continue;
    const int pages = p.pages_of(len);
    const int* from = row(a.forks[2 * i]);
    int* to = row(a.forks[2 * i + 1]);
    int at = need[i];
    for (int b = 0; b < pages; b += 64) {
      const int e = b + lane;
      const int page = e < pages ? from[e] : -1;
      const bool real = e < pages && p.in_pool(page);
      const unsigned long long all = __ballot(real);
      const int r = at + __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(all >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(all), 0));
      if (real) {
        a.src[r] = page;
        a.rows[r] = min(ps, len - e * ps);
      }
      if (e < pages) to[e] = real ? a.dst[r] : page;
      at += __popcll(all);
    }
  }
}

constexpr int kEntries = 1024;  // table entries a workgroup of 256 handles

// Workgroups [0, copy_blocks) copy the pages of the plan; the others (share
// only) each give kEntries of a child's table row the parent's pages, counted once more.
__global__ __launch_bounds__(256) void fork_apply_kernel(ForkArgs a, int copy_blocks, int parts) {
  const Pool& p = a.pool;
  const int b = blockIdx.x;
  if (b < copy_blocks) {
    copy_pages(p, Copies{a.src, a.dst, a.rows, a.count}, b, copy_blocks);
    return;
  }
  const int i = (b - copy_blocks) / parts, part = (b - copy_blocks) % parts;
  const int len = a.len[i];
  if (len < 0) return;
  const int whole = len / p.page_size, pages = p.pages_of(len);
  const int* from = p.table + static_cast<long long>(a.forks[2 * i]) * p.max_pages;
  int* to = p.table + static_cast<long long>(a.forks[2 * i + 1]) * p.max_pages;
  for (int e = part * kEntries + threadIdx.x; e < min(pages, (part + 1) * kEntries); e += 256) {
    const int page = from[e];
    if (e < whole) {
      to[e] = page;
      if (p.in_pool(page)) atomicAdd(p.refs + page, 1);
    } else {
      to[e] = p.in_pool(page) ? a.dst[a.first[i]] : page;
    }
  }
}

// ----------------------------------------------------------------- compact ----
constexpr int kSegment = 4096;  // pages a workgroup of 256 counts

struct CompactArgs {
  Pool pool;
  int* moved;   // (1)
  int* counts;  // workspace (segments): pages in use
  int* src;     // workspace (num_pages / 2 + 1): pages in use at or above their number, ascending
  int* dst;     // workspace (num_pages / 2 + 1): free pages below it, ascending
  int* rank;    // workspace (num_pages, to a multiple of 4): index into src of a page at or above it, or -1
  int* head;    // workspace (2): pages to move, pages in use
  int segments;
};

// Bit j: page base + j is in use (pages past the pool are not).
__device__ __forceinline__ unsigned used_mask(const int* refs, int base, int num_pages) {
  unsigned m = 0;
  if (base + 16 <= num_pages) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int4 r = *reinterpret_cast<const int4*>(refs + base + 4 * j);
      m |= (static_cast<unsigned>(r.x != 0) | static_cast<unsigned>(r.y != 0) << 1 |
            static_cast<unsigned>(r.z != 0) << 2 | static_cast<unsigned>(r.w != 0) << 3) << (4 * j);
    }
  } else {
    for (int j = 0; j < 16; ++j)
      if (base + j < num_pages && refs[base + j] != 0) m |= 1u << j;
  }
  return m;
}

__global__ __launch_bounds__(256) void compact_count_kernel(CompactArgs a) {
  __shared__ int tmp[4];
  int total;
  block_scan<256>(static_cast<int>(__popc(used_mask(a.pool.refs, blockIdx.x * kSegment + threadIdx.x * 16, a.pool.num_pages))), tmp, total);
  if (threadIdx.x == 0) a.counts[blockIdx.x] = total;
}

// Lists pages b .. b + 15 (mask m: those in use; `at`: pages in use before them).
__device__ __forceinline__ void list_pages(const CompactArgs& a, unsigned m, int b, int at, int used, int below) {
  const int P = a.pool.num_pages;
  int rank[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const bool live = m >> j & 1, high = b + j >= used;
    rank[j] = live && high ? at - below : -1;
    if (b + j < P) {
      if (live && high) a.src[at - below] = b + j;
      if (!live && !high) a.dst[b + j - at] = b + j;
    }
    at += live;
  }
  if (b + 16 > used)  // ranks of lower pages are not asked for
    for (int j = 0; j < 16; j += 4)
      if (b + j < P) *reinterpret_cast<int4*>(a.rank + b + j) = make_int4(rank[j], rank[j + 1], rank[j + 2], rank[j + 3]);
}

// With L pages in use, those at or above page L go to the free ones below it,
// both in ascending order: as few moves as there can be, and a source is never
// a destination.
__global__ __launch_bounds__(256) void compact_list_kernel(CompactArgs a) {
  __shared__ long long tmp[4];
  const int P = a.pool.num_pages, seg = blockIdx.x;
  const int b = seg * kSegment + threadIdx.x * 16;
  const unsigned m = used_mask(a.pool.refs, b, P);
  // two sums at a time, in the halves of one: all pages in use (below 2^28), and those of the segments before this one
  long long x = 0, sums;
  for (int i = threadIdx.x; i < a.segments; i += 256) {
    const int c = a.counts[i];
    x += static_cast<long long>(c) << 32 | (i < seg ? c : 0);
  }
  block_scan<256>(x, tmp, sums);
  const int used = static_cast<int>(sums >> 32), before = static_cast<int>(sums & 0xffffffff);
  const int cut = used / kSegment;  // the segment of page `used`
  int under = 0;
  for (int i = threadIdx.x; i < cut; i += 256) under += a.counts[i];
  const int cb = cut * kSegment + threadIdx.x * 16;
  const int inside = min(max(used - cb, 0), 16);
  under += __popc(used_mask(a.pool.refs, cb, P) & ((1u << inside) - 1));
  x = block_scan<256>(static_cast<long long>(under) << 32 | static_cast<long long>(__popc(m)), tmp, sums);
  const int below = static_cast<int>(sums >> 32);                          // pages in use below page `used`
  int at = before + static_cast<int>(x & 0xffffffff);                      // pages in use before page b + j
  if (seg == 0 && threadIdx.x == 0) {
    a.head[0] = used - below;
    a.head[1] = used;
    a.moved[0] = used - below;
  }
  list_pages(a, m, b, at, used, below);
}

// Count and list in one launch of one workgroup, 16 pages to a thread: for pools
// of up to 16384 pages (4,436 pages, few moves, whole call: 11.7 us against 13.7
// with two launches; four rounds of it at 62,000 pages 21.7 against 15.8).
constexpr int kPlanPages = kPlan * 16;

__global__ __launch_bounds__(kPlan) void compact_plan_kernel(CompactArgs a) {
  __shared__ int tmp[kPlan / 64];
  const int b = threadIdx.x * 16;
  const unsigned m = used_mask(a.pool.refs, b, a.pool.num_pages);
  int used, below;
  const int at = block_scan<kPlan>(static_cast<int>(__popc(m)), tmp, used);
  const int inside = min(max(used - b, 0), 16);
  block_scan<kPlan>(static_cast<int>(__popc(m & ((1u << inside) - 1))), tmp, below);  // pages in use below page `used`
  if (threadIdx.x == 0) {
    a.head[0] = used - below;
    a.head[1] = used;
    a.moved[0] = used - below;
  }
  if (used > below) list_pages(a, m, b, at, used, below);
}

// Workgroups [0, copy_blocks) move the pages; the others each rename the pages
// in kEntries of a table row, and between them move the counts.
__global__ __launch_bounds__(256) void compact_move_kernel(CompactArgs a, int copy_blocks, int parts) {
  const Pool& p = a.pool;
  const int moves = a.head[0];
  if (moves == 0) return;
  const int b = blockIdx.x;
  if (b < copy_blocks) {
    copy_pages(p, Copies{a.src, a.dst, nullptr, a.head}, b, copy_blocks);
    return;
  }
  const int used = a.head[1];
  const int t = b - copy_blocks, s = t / parts, part = t % parts;
  for (int k = t * 256 + threadIdx.x; k < moves; k += (gridDim.x - copy_blocks) * 256) {
    p.refs[a.dst[k]] = p.refs[a.src[k]];
    p.refs[a.src[k]] = 0;
  }
  const int len = p.lens[s];
  const int pages = p.len_fits(len) ? p.pages_of(len) : 0;
  int* row = p.table + static_cast<long long>(s) * p.max_pages;
  for (int e = part * kEntries + threadIdx.x; e < min(pages, (part + 1) * kEntries); e += 256) {
    const int page = row[e];
    if (!p.in_pool(page) || page < used) continue;
    const int k = a.rank[page];
    if (k >= 0) row[e] = a.dst[k];
  }
}

// -------------------------------------------------------------------- free ----
constexpr int kFreeEntries = 2048;  // table entries a workgroup of 256 handles

struct FreeArgs {
  Pool pool;
  const int* slots;
  int* status;
  int parts;  // workgroups to a slot
};

// The sequence that entry i of the list ends, or -1: it names none, or one that an earlier entry names.
__device__ __forceinline__ int ended(const FreeArgs& a, int i, int& len) {
  const int s = a.slots[i];
  const bool real = static_cast<unsigned>(s) < static_cast<unsigned>(a.pool.num_seqs);
  len = real ? a.pool.lens[s] : -1;
  bool again = false;
  for (int j = threadIdx.x; j < i; j += 256) again |= a.slots[j] == s;
  return __syncthreads_or(again) || !a.pool.len_fits(len) ? -1 : s;
}

__device__ __forceinline__ void end_slot(const FreeArgs& a, int i, int s) {
  a.status[i] = s < 0 ? PAGE_INVALID : PAGE_DONE;
  if (s >= 0) a.pool.lens[s] = 0;
}

// Part y of slot x's table entries: one round trip for the entries and one for
// their counts. Bound by random 4-byte reads and writes: 355,000 pages all over
// the pool, one in six of them shared, 15.5 us (with the tables put back, in a
// graph: 24, 19 without the atomics, 15 without any write of a count).
// With one part to a slot the length goes to 0 here (the barrier in ended() is
// behind every read of it); with more a second launch does that, as the other
// parts may not have read it yet.
__global__ __launch_bounds__(256) void free_kernel(FreeArgs a) {
  const Pool& p = a.pool;
  const int i = blockIdx.x;
  int len;
  const int s = ended(a, i, len);
  if (a.parts == 1 && threadIdx.x == 0) end_slot(a, i, s);
  if (s < 0) return;
  int* row = p.table + static_cast<long long>(s) * p.max_pages;
  const int pages = p.pages_of(len), e0 = blockIdx.y * kFreeEntries + threadIdx.x;
  int page[kFreeEntries / 256], refs[kFreeEntries / 256];
#pragma unroll
  for (int k = 0; k < kFreeEntries / 256; ++k) page[k] = e0 + 256 * k < pages ? row[e0 + 256 * k] : -1;
#pragma unroll
  for (int k = 0; k < kFreeEntries / 256; ++k) refs[k] = p.in_pool(page[k]) ? p.refs[page[k]] : 0;
#pragma unroll
  for (int k = 0; k < kFreeEntries / 256; ++k) {
    if (e0 + 256 * k < pages) row[e0 + 256 * k] = -1;
    // A page whose count is 1 is held here alone: nobody else changes it. A count
    // that was read too early is too high, and the others' are taken off atomically;
    // one that said too little stays at 0.
    if (refs[k] == 1)
      p.refs[page[k]] = 0;
    else if (refs[k] > 1 && atomicSub(p.refs + page[k], 1) <= 0)
      atomicMax(p.refs + page[k], 0);
  }
}

__global__ __launch_bounds__(256) void free_lens_kernel(FreeArgs a) {
  int len;
  const int s = ended(a, blockIdx.x, len);
  if (threadIdx.x == 0) end_slot(a, blockIdx.x, s);
}

// -------------------------------------------------------------------- host ----
constexpr int kMaxPoolPages = 1 << 27;
constexpr int kCopyBlocks = 2048;

long long round4(long long n) { return (n + 3) / 4 * 4; }

int check_table(const char* who, const void* table, const void* lens, int num_pages, int page_size, int num_seqs, int max_pages) {
  IRON_REQUIRE(table && lens, "%s: null pointer", who);
  for (const void* q : {table, lens})
    IRON_REQUIRE((reinterpret_cast<uintptr_t>(q) & 3u) == 0, "%s: int32 arrays must be 4-byte aligned", who);
  IRON_REQUIRE(num_pages >= 1 && num_pages <= kMaxPoolPages, "%s: num_pages=%d outside [1, %d]", who, num_pages, kMaxPoolPages);
  IRON_REQUIRE(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0,
               "%s: page_size=%d is not a power of two from 16 to 1024", who, page_size);
  IRON_REQUIRE(num_seqs >= 1 && num_seqs <= kMaxSeqs, "%s: num_seqs=%d outside [1, %d]", who, num_seqs, kMaxSeqs);
  IRON_REQUIRE(max_pages >= 1 && static_cast<long long>(max_pages) * page_size < (1LL << 31) - (1 << 20),
               "%s: max_pages=%d: a sequence holds less than 2^31 - 2^20 positions", who, max_pages);
  return 0;
}

int check_pool(const char* who, const void* table, const void* lens, const void* refs, const void* status, int num_pages,
               int page_size, int num_seqs, int max_pages) {
  IRON_REQUIRE(refs && status, "%s: null pointer", who);
  for (const void* q : {refs, status})
    IRON_REQUIRE((reinterpret_cast<uintptr_t>(q) & 3u) == 0, "%s: int32 arrays must be 4-byte aligned", who);
  IRON_REQUIRE(aligned16(refs), "%s: page_refs must be 16-byte aligned", who);
  return check_table(who, table, lens, num_pages, page_size, num_seqs, max_pages);
}

int check_data(const char* who, const void* k, const void* v, int num_layers, int n_kv_heads, int row_bytes) {
  IRON_REQUIRE(k && v, "%s: null pointer", who);
  IRON_REQUIRE(k != v, "%s: k_pages and v_pages are the same buffer", who);
  IRON_REQUIRE(aligned16(k) && aligned16(v), "%s: k_pages and v_pages must be 16-byte aligned", who);
  IRON_REQUIRE(num_layers >= 1 && num_layers <= 1024, "%s: num_layers=%d outside [1, 1024]", who, num_layers);
  IRON_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 1024, "%s: n_kv_heads=%d outside [1, 1024]", who, n_kv_heads);
  IRON_REQUIRE(row_bytes >= 16 && row_bytes <= 4096 && row_bytes % 16 == 0,
               "%s: rows of %d bytes: a multiple of 16 up to 4096 is needed", who, row_bytes);
  return 0;
}

int check_workspace(const char* who, const void* ws, long long bytes, long long need) {
  IRON_REQUIRE(ws && aligned16(ws), "%s: the workspace must be given and 16-byte aligned", who);
  IRON_REQUIRE(bytes >= need, "%s: workspace of %lld bytes, %lld needed", who, bytes, need);
  return 0;
}

Pool make_pool(void* k, void* v, void* table, void* lens, void* refs, int num_layers, int n_kv_heads, int row_bytes,
               int num_pages, int page_size, int num_seqs, int max_pages) {
  Pool p;
  p.k = static_cast<unsigned char*>(k);
  p.v = static_cast<unsigned char*>(v);
  p.table = static_cast<int*>(table);
  p.lens = static_cast<int*>(lens);
  p.refs = static_cast<int*>(refs);
  p.num_layers = num_layers;
  p.num_pages = num_pages;
  p.page_size = page_size;
  p.num_seqs = num_seqs;
  p.max_pages = max_pages;
  p.n_kv_heads = n_kv_heads;
  p.row_chunks = row_bytes / 16;
  return p;
}

long long append_list(int num_seqs, int num_rows, int page_size) { return num_rows / page_size + num_seqs; }

// Checks an append and fills its arguments.
int append_call(const char* who, AppendArgs& a, const void* k_new, const void* v_new, const int* rows, const int* row_starts,
                void* k_pages, void* v_pages, int* page_table, int* seq_lens, int* page_refs, int* status, int num_layers,
                int n_kv_heads, int row_bytes, int num_pages, int page_size, int num_seqs, int max_pages, int num_nodes,
                int num_rows, void* workspace, long long workspace_bytes) {
  if (int rc = check_pool(who, page_table, seq_lens, page_refs, status, num_pages, page_size, num_seqs, max_pages)) return rc;
  if (int rc = check_data(who, k_pages, v_pages, num_layers, n_kv_heads, row_bytes)) return rc;
  IRON_REQUIRE(k_new && v_new && rows && row_starts, "%s: null pointer", who);
  IRON_REQUIRE(aligned16(k_new) && aligned16(v_new), "%s: k_new and v_new must be 16-byte aligned", who);
  IRON_REQUIRE(((reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(row_starts)) & 3u) == 0,
               "%s: int32 arrays must be 4-byte aligned", who);
  IRON_REQUIRE(num_nodes >= 1, "%s: num_nodes=%d", who, num_nodes);
  IRON_REQUIRE(num_rows >= 1 && num_rows <= kMaxRows, "%s: num_rows=%d outside [1, %d]", who, num_rows, kMaxRows);
  if (int rc = check_workspace(who, workspace, workspace_bytes,
                               iron_paged_append_workspace_bytes(num_seqs, num_rows, page_size)))
    return rc;
  a.pool = make_pool(k_pages, v_pages, page_table, seq_lens, page_refs, num_layers, n_kv_heads, row_bytes, num_pages,
                     page_size, num_seqs, max_pages);
  a.k_new = static_cast<const uint4*>(k_new);
  a.v_new = static_cast<const uint4*>(v_new);
  a.rows = rows;
  a.row_starts = row_starts;
  a.status = status;
  a.begin = static_cast<int*>(workspace);
  a.list = a.begin + round4(num_seqs);
  a.num_nodes = num_nodes;
  a.num_rows = num_rows;
  a.list_cap = static_cast<int>(append_list(num_seqs, num_rows, page_size));
  return 0;
}

int check_int4(const char* who, int dtype, int head_dim) {
  IRON_REQUIRE(dtype == 0 || dtype == 1, "%s: dtype=%d is neither 0 (bf16) nor 1 (fp16)", who, dtype);
  IRON_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim must be 64 or 128", who);
  return 0;
}

long long fork_list(int num_forks, int max_pages, int num_pages, int share) {
  return share ? num_forks : std::min<long long>(static_cast<long long>(num_forks) * max_pages, num_pages);
}

}  // namespace
}  // namespace iron

using namespace iron;

extern "C" long long iron_paged_append_workspace_bytes(int num_seqs, int num_rows, int page_size) {
  if (num_seqs < 1 || num_seqs > kMaxSeqs || num_rows < 1 || num_rows > kMaxRows || page_size < 16) return -1;
  return 4 * (round4(num_seqs) + append_list(num_seqs, num_rows, page_size));
}

extern "C" int iron_paged_append(const void* k_new, const void* v_new, const int* rows, const int* row_starts,
                                 void* k_pages, void* v_pages, int* page_table, int* seq_lens, int* page_refs,
                                 int* status, int num_layers, int n_kv_heads, int row_bytes, int num_pages,
                                 int page_size, int num_seqs, int max_pages, int num_nodes, int num_rows,
                                 void* workspace, long long workspace_bytes, void* stream) {
  AppendArgs a;
  if (int rc = append_call("iron_paged_append", a, k_new, v_new, rows, row_starts, k_pages, v_pages, page_table, seq_lens,
                           page_refs, status, num_layers, n_kv_heads, row_bytes, num_pages, page_size, num_seqs, max_pages,
                           num_nodes, num_rows, workspace, workspace_bytes))
    return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  IRON_LAUNCH(append_plan_kernel, dim3(1), dim3(kPlan), 0, s, a);
  // as many layers to a workgroup as leave 4096 of them
  const int group = std::min(num_layers, std::max(1, static_cast<int>(static_cast<long long>(num_rows) * num_layers / 4096)));
  IRON_LAUNCH(append_rows_kernel, dim3(num_rows, (num_layers + group - 1) / group), dim3(256), 0, s, a, group);
  return check_launch("paged_append");
}

extern "C" int iron_paged_append_int4(const void* k_new, const void* v_new, const int* rows, const int* row_starts,
                                      void* k_pages, void* v_pages, int* page_table, int* seq_lens, int* page_refs,
                                      int* status, int dtype, int num_layers, int n_kv_heads, int head_dim, int num_pages,
                                      int page_size, int num_seqs, int max_pages, int num_nodes, int num_rows,
                                      void* workspace, long long workspace_bytes, void* stream) {
  const char* who = "iron_paged_append_int4";
  if (int rc = check_int4(who, dtype, head_dim)) return rc;
  AppendArgs a;
  if (int rc = append_call(who, a, k_new, v_new, rows, row_starts, k_pages, v_pages, page_table, seq_lens, page_refs, status,
                           num_layers, n_kv_heads, head_dim / 2 + 16, num_pages, page_size, num_seqs, max_pages, num_nodes,
                           num_rows, workspace, workspace_bytes))
    return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  IRON_LAUNCH(append_plan_kernel, dim3(1), dim3(kPlan), 0, s, a);
  const int planes = num_layers * 2 * n_kv_heads, items = planes_of(num_rows, planes);
  const dim3 grid((num_rows + kTile - 1) / kTile, (planes + items - 1) / items);
  if (head_dim == 64 && dtype)
    IRON_LAUNCH((append4_rows_kernel<64, true>), grid, dim3(256), 0, s, a, items);
  else if (head_dim == 64)
    IRON_LAUNCH((append4_rows_kernel<64, false>), grid, dim3(256), 0, s, a, items);
  else if (dtype)
    IRON_LAUNCH((append4_rows_kernel<128, true>), grid, dim3(256), 0, s, a, items);
  else
    IRON_LAUNCH((append4_rows_kernel<128, false>), grid, dim3(256), 0, s, a, items);
  return check_launch("paged_append_int4");
}

extern "C" int iron_paged_gather_int4(const int* begins, const int* row_starts, const void* k_pages, const void* v_pages,
                                      const int* page_table, const int* seq_lens, void* k_out, void* v_out, int dtype,
                                      int num_layers, int n_kv_heads, int head_dim, int num_pages, int page_size,
                                      int num_seqs, int max_pages, int num_rows, void* stream) {
  const char* who = "iron_paged_gather_int4";
  if (int rc = check_int4(who, dtype, head_dim)) return rc;
  if (int rc = check_table(who, page_table, seq_lens, num_pages, page_size, num_seqs, max_pages)) return rc;
  if (int rc = check_data(who, k_pages, v_pages, num_layers, n_kv_heads, head_dim / 2 + 16)) return rc;
  for (const int* p : {begins, row_starts})
    IRON_REQUIRE(p && (reinterpret_cast<uintptr_t>(p) & 3u) == 0, "%s: int32 arrays must be given and 4-byte aligned", who);
  IRON_REQUIRE(k_out && v_out && aligned16(k_out) && aligned16(v_out), "%s: k_out and v_out must be given and 16-byte aligned", who);
  for (const void* p : {k_pages, v_pages}) IRON_REQUIRE(k_out != p && v_out != p, "%s: k_out or v_out is one of the inputs", who);
  IRON_REQUIRE(k_out != v_out, "%s: k_out and v_out are the same buffer", who);
  IRON_REQUIRE(num_rows >= 1 && num_rows <= kMaxRows, "%s: num_rows=%d outside [1, %d]", who, num_rows, kMaxRows);
  GatherArgs a;
  a.pool = make_pool(const_cast<void*>(k_pages), const_cast<void*>(v_pages), const_cast<int*>(page_table), const_cast<int*>(seq_lens),
                     nullptr, num_layers, n_kv_heads, head_dim / 2 + 16, num_pages, page_size, num_seqs, max_pages);
  a.begins = begins;
  a.row_starts = row_starts;
  a.k_out = static_cast<uint4*>(k_out);
  a.v_out = static_cast<uint4*>(v_out);
  a.num_rows = num_rows;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int planes = num_layers * 2 * n_kv_heads, items = planes_of(num_rows, planes);
  const dim3 grid((num_rows + kTile - 1) / kTile, (planes + items - 1) / items);
  if (head_dim == 64 && dtype)
    IRON_LAUNCH((gather4_rows_kernel<64, true>), grid, dim3(256), 0, s, a, items);
  else if (head_dim == 64)
    IRON_LAUNCH((gather4_rows_kernel<64, false>), grid, dim3(256), 0, s, a, items);
  else if (dtype)
    IRON_LAUNCH((gather4_rows_kernel<128, true>), grid, dim3(256), 0, s, a, items);
  else
    IRON_LAUNCH((gather4_rows_kernel<128, false>), grid, dim3(256), 0, s, a, items);
  return check_launch("paged_gather_int4");
}

extern "C" long long iron_page_fork_workspace_bytes(int num_forks, int num_seqs, int max_pages, int num_pages, int share) {
  if (num_forks < 1 || num_forks > kMaxRequests || num_seqs < 1 || max_pages < 1 || num_pages < 1) return -1;
  return 4 * (4 + 2 * round4(num_forks) + 3 * round4(fork_list(num_forks, max_pages, num_pages, share)));
}

extern "C" int iron_page_fork(const int* forks, void* k_pages, void* v_pages, int* page_table, int* seq_lens,
                              int* page_refs, int* status, int num_layers, int n_kv_heads, int row_bytes, int num_pages,
                              int page_size, int num_seqs, int max_pages, int num_forks, int share, void* workspace,
                              long long workspace_bytes, void* stream) {
  const char* who = "iron_page_fork";
  if (int rc = check_pool(who, page_table, seq_lens, page_refs, status, num_pages, page_size, num_seqs, max_pages)) return rc;
  if (int rc = check_data(who, k_pages, v_pages, num_layers, n_kv_heads, row_bytes)) return rc;
  IRON_REQUIRE(forks && (reinterpret_cast<uintptr_t>(forks) & 3u) == 0, "%s: forks must be given and 4-byte aligned", who);
  IRON_REQUIRE(num_forks >= 1 && num_forks <= kMaxRequests, "%s: num_forks=%d outside [1, %d]", who, num_forks, kMaxRequests);
  IRON_REQUIRE(static_cast<long long>(num_forks) * max_pages < (1LL << 31), "%s: num_forks * max_pages exceeds 2^31", who);
  if (int rc = check_workspace(who, workspace, workspace_bytes,
                               iron_page_fork_workspace_bytes(num_forks, num_seqs, max_pages, num_pages, share)))
    return rc;
  ForkArgs a;
  a.pool = make_pool(k_pages, v_pages, page_table, seq_lens, page_refs, num_layers, n_kv_heads, row_bytes, num_pages,
                     page_size, num_seqs, max_pages);
  const long long cap = fork_list(num_forks, max_pages, num_pages, share);
  a.forks = forks;
  a.status = status;
  a.count = static_cast<int*>(workspace);
  a.len = a.count + 4;
  a.first = a.len + round4(num_forks);
  a.dst = a.first + round4(num_forks);
  a.src = a.dst + round4(cap);
  a.rows = a.src + round4(cap);
  a.num_forks = num_forks;
  a.list_cap = static_cast<int>(cap);
  a.share = share != 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  IRON_LAUNCH(fork_plan_kernel, dim3(1), dim3(kPlan), 0, s, a);
  const int copy_blocks = static_cast<int>(std::min<long long>(kCopyBlocks, cap * num_layers * 2));
  const int parts = (max_pages + kEntries - 1) / kEntries;
  const int blocks = copy_blocks + (share ? num_forks * parts : 0);
  IRON_LAUNCH(fork_apply_kernel, dim3(blocks), dim3(256), 0, s, a, copy_blocks, parts);
  return check_launch("page_fork");
}

extern "C" long long iron_page_compact_workspace_bytes(int num_pages) {
  if (num_pages < 1 || num_pages > kMaxPoolPages) return -1;
  return 4 * (4 + round4((num_pages + kSegment - 1) / kSegment) + 2 * round4(num_pages / 2 + 1) + round4(num_pages));
}

extern "C" int iron_page_compact(void* k_pages, void* v_pages, int* page_table, int* seq_lens, int* page_refs, int* moved,
                                 int num_layers, int n_kv_heads, int row_bytes, int num_pages, int page_size,
                                 int num_seqs, int max_pages, void* workspace, long long workspace_bytes, void* stream) {
  const char* who = "iron_page_compact";
  if (int rc = check_pool(who, page_table, seq_lens, page_refs, moved, num_pages, page_size, num_seqs, max_pages)) return rc;
  if (int rc = check_data(who, k_pages, v_pages, num_layers, n_kv_heads, row_bytes)) return rc;
  if (int rc = check_workspace(who, workspace, workspace_bytes, iron_page_compact_workspace_bytes(num_pages))) return rc;
  const int parts = (max_pages + kEntries - 1) / kEntries;
  IRON_REQUIRE(static_cast<long long>(num_seqs) * parts < (1 << 23), "%s: num_seqs=%d with max_pages=%d: a table of up to 2^33 entries", who,
               num_seqs, max_pages);
  CompactArgs a;
  a.pool = make_pool(k_pages, v_pages, page_table, seq_lens, page_refs, num_layers, n_kv_heads, row_bytes, num_pages,
                     page_size, num_seqs, max_pages);
  a.segments = (num_pages + kSegment - 1) / kSegment;
  a.moved = moved;
  a.head = static_cast<int*>(workspace);
  a.counts = a.head + 4;
  a.src = a.counts + round4(a.segments);
  a.dst = a.src + round4(num_pages / 2 + 1);
  a.rank = a.dst + round4(num_pages / 2 + 1);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (num_pages <= kPlanPages) {
    IRON_LAUNCH(compact_plan_kernel, dim3(1), dim3(kPlan), 0, s, a);
  } else {
    IRON_LAUNCH(compact_count_kernel, dim3(a.segments), dim3(256), 0, s, a);
    IRON_LAUNCH(compact_list_kernel, dim3(a.segments), dim3(256), 0, s, a);
  }
  const int copy_blocks = static_cast<int>(std::min<long long>(kCopyBlocks, static_cast<long long>(num_pages) * num_layers));
  IRON_LAUNCH(compact_move_kernel, dim3(copy_blocks + num_seqs * parts), dim3(256), 0, s, a, copy_blocks, parts);
  return check_launch("page_compact");
}

extern "C" int iron_page_free(const int* slots, int* page_table, int* seq_lens, int* page_refs, int* status,
                              int num_pages, int page_size, int num_seqs, int max_pages, int num_slots, void* stream) {
  const char* who = "iron_page_free";
  if (int rc = check_pool(who, page_table, seq_lens, page_refs, status, num_pages, page_size, num_seqs, max_pages)) return rc;
  IRON_REQUIRE(slots && (reinterpret_cast<uintptr_t>(slots) & 3u) == 0, "%s: slots must be given and 4-byte aligned", who);
  IRON_REQUIRE(num_slots >= 1 && num_slots <= kMaxRequests, "%s: num_slots=%d outside [1, %d]", who, num_slots, kMaxRequests);
  FreeArgs a;
  a.pool = make_pool(nullptr, nullptr, page_table, seq_lens, page_refs, 0, 0, 16, num_pages, page_size, num_seqs, max_pages);
  a.slots = slots;
  a.status = status;
  a.parts = (max_pages + kFreeEntries - 1) / kFreeEntries;
  IRON_REQUIRE(a.parts <= 65535, "%s: max_pages=%d: at most %d table entries to a sequence", who, max_pages, 65535 * kFreeEntries);
  hipStream_t s = static_cast<hipStream_t>(stream);
  IRON_LAUNCH(free_kernel, dim3(num_slots, a.parts), dim3(256), 0, s, a);
  if (a.parts > 1) IRON_LAUNCH(free_lens_kernel, dim3(num_slots), dim3(256), 0, s, a);
  return check_launch("page_free");
}
