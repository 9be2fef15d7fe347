// Rows of tables of states: copied, cleared, and gathered in front.
//
//   copy      table[target[i]] = table[source[i]] for all pairs i, all rows read before one is written, so that rows may change places
//   clear     table[row] = 0
//   compact   n rows in use: the k-th used row from n on moves to the k-th free row in front of n, which is the least that has to move
//
// Bound by memory: a row is read and written once.  A CTA has a slab of neighbouring bytes of all rows of a table: what it reads and writes no
// other CTA touches, so that "read before written" is a barrier, not a second launch and a copy in between.  A copy's rows pass through
// shared memory, all pairs of them; a compaction reads what it never writes, and goes through registers.
//
// Measured: 64 of 256 rows of 1.6 MB moved in 34.4 us (5.9 TB/s), copied in 42.6 us (4.8 TB/s; the pairs are read and told apart by every CTA); 8 rows of
// 143 KB written in 2.1 us, a launch.
#include <algorithm>

#include "ttt_elem.cuh"

namespace {

using namespace ttt;

constexpr int kThreads = 256;
constexpr int kMost = TTT_B200_TABLES;
constexpr int kMarked = 8192;       // rows that a CTA can mark in shared memory

struct Tables {
  char* base[kMost];
  int64_t units[kMost];      // of a row
  int first[kMost + 1];      // CTA of a table
  int shift;                 // 2^shift units of a row that a CTA has
  int count, rows, pairs;
  int marks;                 // a copy's with more rows than a CTA marks: 2^marks places, at least twice as many as pairs; else -1
  const int32_t *source, *target;
  const uint8_t* used;
  int32_t* place;
};

// what a CTA works on
template <class U> struct Slab {
  U* base;          // its first unit of row 0
  int64_t row;      // units from row to row
  int n;            // units of a row that there are
  __device__ __forceinline__ explicit Slab(const Tables& q) {
    int k = 0;
    while (static_cast<int>(blockIdx.x) >= q.first[k + 1]) ++k;
    const int64_t at = static_cast<int64_t>(blockIdx.x - q.first[k]) << q.shift;
    base = reinterpret_cast<U*>(q.base[k]) + at;
    row = q.units[k];
    n = static_cast<int>(min(int64_t{1} << q.shift, row - at));
  }
};

// A row that two pairs name as their target gets the later one's: each target has its last pair in shared memory.  Where a CTA can mark all rows, a row's
// place there is its number.  With more rows it is its number's hash, among at least twice as many places as pairs, and the next one where another row has that: 4096
// pairs of 8193 rows of 4 KB 71 us, for 2645 with a search of the pairs behind each; of 8192 rows 71 as well, for 37 with a place for each row.
__device__ __forceinline__ uint32_t place_of(uint32_t row, int bits) {
  row *= 0x9e3779b1u;
  row ^= row >> 15;
  return row * 0x9e3779b1u >> (32 - bits);
}
__device__ __forceinline__ bool inside(const Tables& q, int i) {
  return static_cast<uint32_t>(q.target[i]) < static_cast<uint32_t>(q.rows) && static_cast<uint32_t>(q.source[i]) < static_cast<uint32_t>(q.rows);
}

template <class U> __global__ void __launch_bounds__(kThreads) copy_rows_kernel(const Tables q) {
  wait_for_predecessor();
  extern __shared__ __align__(16) unsigned char memory[];
  const Slab<U> s(q);
  int32_t* from = reinterpret_cast<int32_t*>(memory);      // of a pair that is taken: its rows; else -1
  int32_t* to = from + q.pairs;
  int32_t* last = to + q.pairs;                            // of a place: its row's last pair
  const bool hashed = q.marks >= 0;
  const int places = hashed ? 1 << q.marks : q.rows;
  int32_t* row = last + places;                            // hashed: and that row
  for (int k = threadIdx.x; k < places; k += kThreads) {
    last[k] = -1;
    if (hashed) row[k] = -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < q.pairs; i += kThreads) {
    if (!inside(q, i)) continue;
    const int t = q.target[i];
    uint32_t k = t;
    if (hashed) {
      k = place_of(t, q.marks);
      for (int tries = 0; tries < places; ++tries, k = (k + 1) & (places - 1)) {      // (half of the places stay free)
        const int32_t who = atomicCAS(&row[k], -1, t);
        if (who == -1 || who == t) break;
      }
    }
    atomicMax(&last[k], i);      // (a maximum does not go by the order)
  }
  __syncthreads();
  for (int i = threadIdx.x; i < q.pairs; i += kThreads) {
    const int t = q.target[i];
    bool take = inside(q, i);
    if (take) {
      uint32_t k = t;
      if (hashed) {
        k = place_of(t, q.marks);
        for (int tries = 0; tries < places && row[k] != t; ++tries) k = (k + 1) & (places - 1);
      }
      take = last[k] == i;
    }
    from[i] = take ? q.source[i] : -1;
    to[i] = t;
  }
  __syncthreads();
  U* stage = reinterpret_cast<U*>(memory + (8L * q.pairs + (hashed ? 8L : 4L) * places + 15) / 16 * 16);
  const int total = q.pairs << q.shift;
#pragma unroll 4
  for (int k = threadIdx.x; k < total; k += kThreads) {
    const int i = k >> q.shift, u = k & ((1 << q.shift) - 1);
    if (from[i] >= 0 && u < s.n) stage[k] = s.base[from[i] * s.row + u];
  }
  __syncthreads();
  for (int k = threadIdx.x; k < total; k += kThreads) {
    const int i = k >> q.shift, u = k & ((1 << q.shift) - 1);
    if (from[i] >= 0 && u < s.n) s.base[to[i] * s.row + u] = stage[k];
  }
}

template <class U> __global__ void __launch_bounds__(kThreads) clear_rows_kernel(const Tables q) {
  wait_for_predecessor();
  const Slab<U> s(q);
  const U zero = {};
  for (int k = threadIdx.x; k < q.pairs << q.shift; k += kThreads) {
    const int i = k >> q.shift, u = k & ((1 << q.shift) - 1);
    if (static_cast<uint32_t>(q.target[i]) < static_cast<uint32_t>(q.rows) && u < s.n) s.base[q.target[i] * s.row + u] = zero;
  }
}

// How many of the threads in front of this one, and of all of them, say yes.
__device__ __forceinline__ int before(bool yes, int* warps, int& all) {
  const uint32_t votes = __ballot_sync(0xffffffffu, yes);
  const int warp = threadIdx.x / 32;
  __syncthreads();
  if (threadIdx.x % 32 == 0) warps[warp] = __popc(votes);
  __syncthreads();
  int mine = __popc(votes & ((1u << threadIdx.x % 32) - 1));
  all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) mine += warps[w];
    all += warps[w];
  }
  return mine;
}

template <class U> __global__ void __launch_bounds__(kThreads) compact_rows_kernel(const Tables q) {
  wait_for_predecessor();
  extern __shared__ __align__(16) unsigned char memory[];
  __shared__ int warps[kThreads / 32];
  uint16_t* from = reinterpret_cast<uint16_t*>(memory);      // (at most half of the rows move)
  uint16_t* to = from + q.rows / 2 + 1;
  int n = 0;
  for (int r = threadIdx.x; r < q.rows; r += kThreads) n += q.used[r] != 0;
  for (int o = 16; o; o /= 2) n += __shfl_xor_sync(0xffffffffu, n, o);
  if (threadIdx.x % 32 == 0) warps[threadIdx.x / 32] = n;
  __syncthreads();
  n = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) n += warps[w];
  int holes = 0, moves = 0;
  for (int r0 = 0; r0 < q.rows; r0 += kThreads) {
    const int r = r0 + static_cast<int>(threadIdx.x);
    const bool in = r < q.rows, use = in && q.used[r], hole = in && !use && r < n, late = use && r >= n;
    int all;
    const int h = before(hole, warps, all) + holes;
    holes += all;
    const int l = before(late, warps, all) + moves;
    moves += all;
    if (hole) to[h] = static_cast<uint16_t>(r);
    if (late) from[l] = static_cast<uint16_t>(r);
    if (blockIdx.x == 0 && q.place && in && !late) q.place[r] = use ? r : -1;
  }
  __syncthreads();
  if (blockIdx.x == 0 && q.place)
    for (int k = threadIdx.x; k < moves; k += kThreads) q.place[from[k]] = to[k];
  if (static_cast<int>(blockIdx.x) >= q.first[q.count]) return;      // (a launch without tables, for the places)
  const Slab<U> s(q);
  const int total = moves << q.shift;
#pragma unroll 4
  for (int k = threadIdx.x; k < total; k += kThreads) {
    const int i = k >> q.shift, u = k & ((1 << q.shift) - 1);
    if (u < s.n) s.base[to[i] * s.row + u] = s.base[from[i] * s.row + u];
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------
int check(const ttt_b200_tables_args* p) {
  if (!p) return fail("tables: NULL argument struct");
  if (p->count < 0 || p->count > kMost) return fail("tables: at most 16 tables");
  if (p->rows < 1 || p->rows > 1 << 30) return fail("tables: 1 to 2^30 rows");
  for (int k = 0; k < p->count; ++k)
    if (!p->table[k] || p->row_bytes[k] < 1) return fail("tables: a table without a pointer or bytes");
  return TTT_B200_OK;
}

// The largest unit that all rows start on a boundary of, and slabs of as many units as leave several CTAs to an SM, at least 128 bytes of a row where
// there are that many.
int unit_of(const ttt_b200_tables_args& p) {
  uint64_t all = 16;
  for (int k = 0; k < p.count; ++k) all |= static_cast<uint64_t>(p.row_bytes[k]) | reinterpret_cast<uintptr_t>(p.table[k]);
  return static_cast<int>(all & -all);
}
int lay_out(Tables& q, const ttt_b200_tables_args& p, int unit, int64_t most_units) {
  q.count = p.count;
  q.rows = p.rows;
  int64_t all = 0;
  for (int k = 0; k < p.count; ++k) {
    q.base[k] = static_cast<char*>(p.table[k]);
    q.units[k] = p.row_bytes[k] / unit;
    all += q.units[k];
  }
  const int64_t few = std::max<int64_t>(128 / unit, all / (4L * sm_count()));
  const int64_t want = std::min<int64_t>({few, 4096 / unit, most_units});
  while (2L << q.shift <= want) ++q.shift;
  int64_t ctas = 0;
  for (int k = 0; k < p.count; ++k) {
    q.first[k] = static_cast<int>(ctas);
    ctas += ((q.units[k] - 1) >> q.shift) + 1;
    if (ctas > 0x7fffffffL) return fail("tables: rows of too many bytes");
    q.first[k + 1] = static_cast<int>(ctas);
  }
  return TTT_B200_OK;
}

#define TTT_WITH_UNIT(unit, body)                      \
  switch (unit) {                                      \
    case 16: { using U = uint4; body; break; }         \
    case 8: { using U = uint2; body; break; }          \
    case 4: { using U = uint32_t; body; break; }       \
    case 2: { using U = uint16_t; body; break; }       \
    default: { using U = uint8_t; body; break; }       \
  }

template <class U> int copy(const Tables& q, uint32_t bytes, cudaStream_t s) {
  if (int rc = allow_shared<copy_rows_kernel<U>>()) return rc;
  ttt_launch_overlapped(copy_rows_kernel<U>, q.first[q.count], kThreads, bytes, s, q);
  return launched("copy rows");
}

}  // namespace

extern "C" int ttt_b200_copy_rows(const ttt_b200_tables_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (p->pairs < 0 || p->pairs > TTT_B200_TABLE_PAIRS) return fail("copy rows: at most 4096 pairs");
  if (p->pairs == 0 || p->count == 0) return fail("copy rows: nothing to copy");
  if (!p->source || !p->target) return fail("copy rows: null tensor pointer");
  Tables q = {};
  q.pairs = p->pairs;
  q.source = p->source;
  q.target = p->target;
  const int unit = unit_of(*p);
  // shared memory: the pairs, the targets' places, and the slab of every pair: 32 KB, with many pairs as much as 16 bytes of each take
  q.marks = -1;
  if (p->rows > kMarked)
    for (q.marks = 1; 1 << q.marks < 2 * q.pairs;) ++q.marks;
  const int64_t lists = (8L * q.pairs + (q.marks < 0 ? 4L * p->rows : 8L << q.marks) + 15) / 16 * 16;
  const int64_t room = std::max<int64_t>(32 * 1024, 16L * q.pairs);
  if (int rc = lay_out(q, *p, unit, room / (static_cast<int64_t>(unit) * q.pairs))) return rc;
  const uint32_t bytes = static_cast<uint32_t>(lists + (static_cast<int64_t>(unit) * q.pairs << q.shift));
  TTT_WITH_UNIT(unit, return copy<U>(q, bytes, static_cast<cudaStream_t>(stream)))
  return TTT_B200_OK;
}

extern "C" int ttt_b200_clear_rows(const ttt_b200_tables_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (p->pairs < 0 || p->pairs > TTT_B200_TABLE_PAIRS) return fail("clear rows: at most 4096 rows");
  if (p->pairs == 0 || p->count == 0) return fail("clear rows: nothing to clear");
  if (!p->target) return fail("clear rows: null tensor pointer");
  Tables q = {};
  q.pairs = p->pairs;
  q.target = p->target;
  const int unit = unit_of(*p);
  if (int rc = lay_out(q, *p, unit, 4096 / unit)) return rc;
  TTT_WITH_UNIT(unit, ttt_launch_overlapped(clear_rows_kernel<U>, q.first[q.count], kThreads, 0, static_cast<cudaStream_t>(stream), q))
  return launched("clear rows");
}

extern "C" int ttt_b200_compact_rows(const ttt_b200_tables_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (p->rows > kMarked) return fail("compact rows: at most 8192 rows");
  if (!p->used || !p->place) return fail("compact rows: null tensor pointer");
  Tables q = {};
  q.used = p->used;
  q.place = p->place;
  const int unit = p->count ? unit_of(*p) : 16;
  if (int rc = lay_out(q, *p, unit, 4096 / unit)) return rc;
  const uint32_t bytes = (p->rows / 2 + 1) * 4;
  TTT_WITH_UNIT(unit, ttt_launch_overlapped(compact_rows_kernel<U>, std::max(1, q.first[q.count]), kThreads, bytes, static_cast<cudaStream_t>(stream), q))
  return launched("compact rows");
}
