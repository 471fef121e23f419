// Page tables of sequences that share pages, and pages copied and moved.
//
// Whole pages of a sequence are never written again, so that sequences that begin alike
// may name the same ones; a page that is filled in part belongs to one sequence.  Which pages
// are in use is read from the tables themselves (a bit for each page of the pool, in
// LDS), not counted along: nothing has to be kept up to date beside the tables.
#include "atf_launch.h"

namespace atf {

constexpr int kPgThreads = 1024;
constexpr int kPgWaves = kPgThreads / 64;

__device__ __forceinline__ int pages_of(int64_t tokens) { return static_cast<int>((tokens + kPage - 1) / kPage); }

// Exclusive sum over the workgroup's threads; `all`: the whole.  part: kPgWaves ints of LDS.
__device__ __forceinline__ int sum_before(int x, int32_t* part, int* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int in = x;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int up = __shfl_up(in, m);
    in += lane >= m ? up : 0;
  }
  __syncthreads();
  if (lane == 63) part[wave] = in;
  __syncthreads();
  int before = in - x, total = 0;
#pragma unroll
  for (int w = 0; w < kPgWaves; ++w) {
    before += w < wave ? part[w] : 0;
    total += part[w];
  }
  *all = total;
  return before;
}

// The words of a bit map of `pages` pages that thread tid scans: first, and how many of a thread
// (odd: the threads' words lie in different LDS banks).
__device__ __forceinline__ int words_of_thread(int words) { return ((words + kPgThreads - 1) / kPgThreads) | 1; }

// f(page) for every entry of the rows that `wanted(row)` names, of the pages of its tokens, by
// the whole workgroup: 256 entries of a row at a time to each wave.
template <class Wanted, class F>
__device__ __forceinline__ void for_entries(const int32_t* table, int max_pages, const int32_t* seq_lens, int batch,
                                            int most, Wanted wanted, F f) {
  const int lane = threadIdx.x & 63, per_row = (most + 255) / 256;
  for (int64_t item = threadIdx.x >> 6; item < static_cast<int64_t>(batch) * per_row; item += kPgWaves) {
    const int b = static_cast<int>(item / per_row), c0 = static_cast<int>(item % per_row) * 256;
    if (!wanted(b)) continue;
    const int have = min(pages_of(max(seq_lens[b], 0)), max_pages);
    const int32_t* row = table + static_cast<int64_t>(b) * max_pages;
    int pg[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + 64 * i + lane;
      pg[i] = c < have ? row[c] : -1;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) f(pg[i]);
  }
}

// LDS past 64 KB in all has to be asked for; the kernels' static part, which comes on top of the
// dynamic one, is 4.2 KB at most.
static hipError_t allow_lds(const void* kernel, size_t bytes) {
  if (bytes <= 56 * 1024) return hipSuccess;
  return hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
}

// New row b of the tables is old row parents[b].
//   The parent's whole pages are named again.  Its last page, where it is filled in part, stays
// with one of its children (itself, or else the lowest); every other child takes a page from
// the end of the free pages, and copy_src, copy_dst name the copy.  Pages that only rows
// without a child named go to the end of the free pages before that, the lowest id first.
//   Latency bound.  Workgroup 0 finds the pages that become free (bits of the dropped rows'
// pages, less the surviving rows'), and hands out the new ones; the others write the new
// rows, all but the entries of new pages.  8 beams of 375 pages 6.4 us, one prompt of 1876 pages
// forked into 48 rows 5.6; 64 rows of 500 pages 15, of 2000 53, half a million entries 190: one
// workgroup reads every entry of the old rows.  Several could, with the bits in memory and another
// launch, which the small tables would pay for.
constexpr int kSelChunk = 4096;  // entries of a row that a workgroup writes
__global__ __launch_bounds__(kPgThreads) void select_tables_kernel(SelectTablesArgs a) {
  extern __shared__ uint32_t sh[];
  __shared__ int32_t part[kPgWaves];
  __shared__ int s_most, s_dropped;
  const int tid = threadIdx.x;
  auto length = [&](int b) { return max(a.seq_lens[b], 0); };
  auto whole = [&](int b) { return min(length(b) / kPage, a.max_pages); };
  auto pages = [&](int b) { return min(pages_of(length(b)), a.max_pages); };
  auto parent = [&](int b) {
    const int p = a.parents[b];
    return p >= 0 && p < a.batch ? p : -1;
  };
  if (blockIdx.x > 0) {  // ---- row b: entries c0 .. ----
    const int b = blockIdx.y, c0 = (blockIdx.x - 1) * kSelChunk;
    const int p = parent(b);
    int n_whole = 0, n = 0;
    bool keep = false;
    if (p >= 0) {
      n_whole = whole(p);
      n = pages(p);
      if (n > n_whole && n_whole >= c0 && n_whole < c0 + kSelChunk) {  // who keeps the last page (uniform)
        if (parent(p) == p) {
          keep = p == b;
        } else {
          int lower = 0;  // children before b
          for (int i = tid; i < b; i += kPgThreads) lower |= a.parents[i] == p ? 1 : 0;
          keep = __syncthreads_or(lower) == 0;
        }
      }
    }
    const int32_t* from = a.page_table + static_cast<int64_t>(max(p, 0)) * a.max_pages;
    int32_t* to = a.table_out + static_cast<int64_t>(b) * a.max_pages;
    for (int c = c0 + tid; c < min(c0 + kSelChunk, a.max_pages); c += kPgThreads) {
      if (c < n_whole) to[c] = from[c];
      else if (c >= n) to[c] = -1;
      else if (keep) to[c] = from[c];
      // (the entry of a new page: workgroup 0)
    }
    return;
  }
  if (blockIdx.y > 0) return;
  // ---- the pages that become free, the new pages ----
  const int words = (a.num_pages + 31) / 32, each = words_of_thread(words);
  int32_t* keeper = reinterpret_cast<int32_t*>(sh);  // [batch] who keeps a row's last page; batch: no child
  uint32_t* bits = sh + a.batch;                     // [words]
  for (int b = tid; b < a.batch; b += kPgThreads) keeper[b] = a.batch;
  if (tid == 0) {
    s_most = 0;
    s_dropped = 0;
  }
  __syncthreads();
  for (int b = tid; b < a.batch; b += kPgThreads) {
    const int p = parent(b);
    if (p >= 0) atomicMin(&keeper[p], p == b ? -1 : b);
    a.lens_out[b] = p >= 0 ? length(p) : 0;
    atomicMax(&s_most, pages(b));
  }
  __syncthreads();
  for (int b = tid; b < a.batch; b += kPgThreads)
    if (keeper[b] == a.batch && pages(b) > 0) s_dropped = 1;
  __syncthreads();
  const int count = min(max(a.free_count[0], 0), a.num_free);
  int freed = 0;
  if (s_dropped) {
    for (int w = tid; w < words; w += kPgThreads) bits[w] = 0;
    __syncthreads();
    for_entries(a.page_table, a.max_pages, a.seq_lens, a.batch, s_most, [&](int b) { return keeper[b] == a.batch; },
                [&](int pg) {
                  if (pg >= 0 && pg < a.num_pages) atomicOr(&bits[pg >> 5], 1u << (pg & 31));
                });
    __syncthreads();
    for_entries(a.page_table, a.max_pages, a.seq_lens, a.batch, s_most, [&](int b) { return keeper[b] != a.batch; },
                [&](int pg) {
                  if (pg >= 0 && pg < a.num_pages) atomicAnd(&bits[pg >> 5], ~(1u << (pg & 31)));
                });
    __syncthreads();
    int mine = 0;
    for (int w = tid * each; w < min((tid + 1) * each, words); ++w) mine += __builtin_popcount(bits[w]);
    int at = count + sum_before(mine, part, &freed);
    for (int w = tid * each; w < min((tid + 1) * each, words); ++w) {
      for (uint32_t m = bits[w]; m != 0; m &= m - 1) {
        if (at < a.num_free) a.free_pages[at] = 32 * w + __builtin_ctz(m);
        ++at;
      }
    }
  }
  const int have = min(count + freed, a.num_free);
  int taken = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kPgThreads) {
    const int b = b0 + tid;
    int last = -1, col = 0, want = 0;
    if (b < a.batch) {
      const int p = parent(b);
      if (p >= 0 && pages(p) > whole(p) && (keeper[p] == -1 ? p : keeper[p]) != b) {
        col = whole(p);
        last = a.page_table[static_cast<int64_t>(p) * a.max_pages + col];
        want = last >= 0 && last < a.num_pages ? 1 : 0;
        if (!want) a.table_out[static_cast<int64_t>(b) * a.max_pages + col] = -1;
      }
    }
    int all = 0;
    const int nth = taken + sum_before(want, part, &all);  // (its barriers: the freed pages are written)
    taken += all;
    if (b < a.batch) {
      int pg = -1;
      if (want) {
        pg = nth < have ? a.free_pages[have - 1 - nth] : -1;
        a.table_out[static_cast<int64_t>(b) * a.max_pages + col] = pg;
      }
      const bool copy = pg >= 0 && pg < a.num_pages;
      a.copy_src[b] = copy ? last : -1;
      a.copy_dst[b] = copy ? pg : -1;
    }
  }
  if (tid == 0) a.free_left[0] = have - taken;
}

hipError_t launch_select_tables(const SelectTablesArgs& a, hipStream_t s) {
  const size_t lds = (static_cast<size_t>(a.batch) + (a.num_pages + 31) / 32) * sizeof(uint32_t);
  if (hipError_t e = allow_lds(reinterpret_cast<const void*>(select_tables_kernel), lds); e != hipSuccess) return e;
  hipLaunchKernelGGL(select_tables_kernel, dim3(1 + (a.max_pages + kSelChunk - 1) / kSelChunk, a.batch), dim3(kPgThreads), lds, s, a);
  return hipGetLastError();
}

// The pages of the rows moved to the lowest ids that rows and free pages have.
//   With L pages in rows, T = the id of the (L + 1)-th lowest page that is in a row or free:
// rows' pages from T on move, free ones below T take them, the i-th highest of the former to
// the i-th lowest of the latter (as many of each).  The free pages come out highest first,
// so that the lowest is taken first.  Latency bound (the pages' copies are not its part).  One
// workgroup: a page's place depends on all before it.  Marking and rewriting the entries do not, and
// large tables would be faster with several workgroups and two launches more.  Pools of 300 pages 9.7 us, 6000 19,
// 160000 183, 2^19 820; the copies of the 6000 move 2.7 GB in 541 us.
__global__ __launch_bounds__(kPgThreads) void compact_tables_kernel(CompactTablesArgs a) {
  extern __shared__ uint32_t sh[];
  __shared__ int32_t part[kPgWaves], before_live[kPgThreads];
  __shared__ int s_most, s_limit;
  const int tid = threadIdx.x;
  const int words = (a.num_pages + 31) / 32, each = words_of_thread(words);
  uint32_t* live = sh;          // pages in rows
  uint32_t* idle = sh + words;  // free pages
  auto pages = [&](int b) { return min(pages_of(max(a.seq_lens[b], 0)), a.max_pages); };
  for (int w = tid; w < 2 * words; w += kPgThreads) sh[w] = 0;
  if (tid == 0) {
    s_most = 0;
    s_limit = a.num_pages;
  }
  __syncthreads();
  for (int b = tid; b < a.batch; b += kPgThreads) atomicMax(&s_most, pages(b));
  const int count = min(max(a.free_count[0], 0), a.num_free);
  for (int i = tid; i < count; i += kPgThreads) {
    const int pg = a.free_pages[i];
    if (pg >= 0 && pg < a.num_pages) atomicOr(&idle[pg >> 5], 1u << (pg & 31));
  }
  __syncthreads();
  for_entries(a.page_table, a.max_pages, a.seq_lens, a.batch, s_most, [](int) { return true; }, [&](int pg) {
    if (pg >= 0 && pg < a.num_pages) atomicOr(&live[pg >> 5], 1u << (pg & 31));
  });
  __syncthreads();
  const int w0 = min(tid * each, words), w1 = min(w0 + each, words);
  int n_live = 0, n_idle = 0;
  for (int w = w0; w < w1; ++w) {
    idle[w] &= ~live[w];  // (a page that rows hold is not free, whatever the list says)
    n_live += __builtin_popcount(live[w]);
    n_idle += __builtin_popcount(idle[w]);
  }
  int all_live = 0, all_idle = 0;
  const int live0 = sum_before(n_live, part, &all_live);
  const int idle0 = sum_before(n_idle, part, &all_idle);
  before_live[tid] = live0;
  if (live0 + idle0 <= all_live && all_live < live0 + idle0 + n_live + n_idle) {  // the (L + 1)-th lies here
    int skip = all_live - live0 - idle0;
    for (int w = w0; w < w1; ++w) {
      uint32_t m = live[w] | idle[w];
      const int n = __builtin_popcount(m);
      if (skip >= n) {
        skip -= n;
        continue;
      }
      for (; skip > 0; --skip) m &= m - 1;
      s_limit = 32 * w + __builtin_ctz(m);
      break;
    }
  }
  __syncthreads();
  const int limit = s_limit;
  int nl = live0, ni = idle0, moves = 0;
  for (int w = w0; w < w1; ++w) {
    for (uint32_t m = live[w] | idle[w]; m != 0; m &= m - 1) {
      const int pg = 32 * w + __builtin_ctz(m);
      const bool is_live = (live[w] >> (pg & 31)) & 1;
      if (is_live && pg >= limit) a.copy_src[all_live - 1 - nl] = pg;
      if (!is_live && pg < limit) {
        a.copy_dst[ni] = pg;
        ++moves;
      }
      if (pg >= limit) a.free_out[all_live + all_idle - 1 - (nl + ni)] = pg;
      nl += is_live ? 1 : 0;
      ni += is_live ? 0 : 1;
    }
  }
  int all_moves = 0;
  sum_before(moves, part, &all_moves);
  for (int i = all_moves + tid; i < a.copies; i += kPgThreads) {
    a.copy_src[i] = -1;
    a.copy_dst[i] = -1;
  }
  for (int i = all_idle + tid; i < a.num_free; i += kPgThreads) a.free_out[i] = -1;
  if (tid == 0) {
    a.free_left[0] = all_idle;
    a.n_copies[0] = all_moves;
  }
  __syncthreads();  // (copy_dst is read below)
  const int64_t entries = static_cast<int64_t>(a.batch) * a.max_pages;
  for (int64_t e = tid; e < entries; e += kPgThreads) {
    const int b = static_cast<int>(e / a.max_pages), c = static_cast<int>(e - static_cast<int64_t>(b) * a.max_pages);
    int pg = c < pages(b) ? a.page_table[e] : -1;
    if (pg >= limit && pg < a.num_pages) {
      const int w = pg >> 5, t = w / each;
      int rank = before_live[t] + __builtin_popcount(live[w] & ((1u << (pg & 31)) - 1));
      for (int u = t * each; u < w; ++u) rank += __builtin_popcount(live[u]);
      pg = a.copy_dst[all_live - 1 - rank];
    }
    a.table_out[e] = pg;
  }
}

hipError_t launch_compact_tables(const CompactTablesArgs& a, hipStream_t s) {
  const size_t lds = 2 * static_cast<size_t>((a.num_pages + 31) / 32) * sizeof(uint32_t);
  if (hipError_t e = allow_lds(reinterpret_cast<const void*>(compact_tables_kernel), lds); e != hipSuccess) return e;
  hipLaunchKernelGGL(compact_tables_kernel, dim3(1), dim3(kPgThreads), lds, s, a);
  return hipGetLastError();
}

// Page dst[i] of every cache becomes a copy of its page src[i].  Bound by HBM: a page's
// bytes read and written; 1500 pages of 28 layers, 2.75 GB, 541 us, 5.1 TB/s.  grid: x = pieces of 16 KB of the pairs' pages, y = cache.
constexpr int kCopyThreads = 256, kCopyUnroll = 4;
constexpr int kCopyPiece = kCopyThreads * kCopyUnroll * 16;

template <typename T>
__device__ __forceinline__ void copy_elements(uint8_t* to, const uint8_t* from, int64_t bytes) {
  for (int64_t i = threadIdx.x; i < bytes / static_cast<int64_t>(sizeof(T)); i += kCopyThreads)
    reinterpret_cast<T*>(to)[i] = reinterpret_cast<const T*>(from)[i];
}

__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(CopyPagesArgs a) {
  const int n = a.count != nullptr ? min(max(a.count[0], 0), a.n) : a.n;
  const int64_t bytes = a.bytes[blockIdx.y];
  uint8_t* base = a.base[blockIdx.y];
  const int64_t pieces = (bytes + kCopyPiece - 1) / kCopyPiece;
  const uint64_t odd = reinterpret_cast<uintptr_t>(base) | static_cast<uint64_t>(bytes);
  for (int64_t item = blockIdx.x; item < n * pieces; item += gridDim.x) {
    const int i = static_cast<int>(item / pieces);
    const int64_t at = (item - i * pieces) * kCopyPiece;
    const int from = a.src[i], to = a.dst[i];
    if (from < 0 || from >= a.num_pages || to < 0 || to >= a.num_pages || from == to) continue;
    const uint8_t* s = base + from * bytes + at;
    uint8_t* d = base + to * bytes + at;
    const int64_t len = min(bytes - at, static_cast<int64_t>(kCopyPiece));
    if ((odd & 15) == 0) {
      u32x4 v[kCopyUnroll];
#pragma unroll
      for (int u = 0; u < kCopyUnroll; ++u) {
        const int64_t o = 16 * static_cast<int64_t>(u * kCopyThreads + threadIdx.x);
        if (o < len) v[u] = ldg16(s + o);
      }
#pragma unroll
      for (int u = 0; u < kCopyUnroll; ++u) {
        const int64_t o = 16 * static_cast<int64_t>(u * kCopyThreads + threadIdx.x);
        if (o < len) *reinterpret_cast<u32x4*>(d + o) = v[u];
      }
    } else if ((odd & 3) == 0) {
      copy_elements<uint32_t>(d, s, len);
    } else {
      copy_elements<uint8_t>(d, s, len);
    }
  }
}

hipError_t launch_copy_pages(const CopyPagesArgs& a, hipStream_t s) {
  if (a.n <= 0 || a.n_caches <= 0) return hipSuccess;
  int64_t most = 1;
  for (int i = 0; i < a.n_caches; ++i) {
    const int64_t p = (a.bytes[i] + kCopyPiece - 1) / kCopyPiece;
    if (p > most) most = p;
  }
  // at most about 16 workgroups a CU: the rest of the pairs in turn
  const int64_t items = a.n * most, cap = (4096 + a.n_caches - 1) / a.n_caches;
  hipLaunchKernelGGL(copy_pages_kernel, dim3(static_cast<unsigned>(items < cap ? items : cap), a.n_caches),
                     dim3(kCopyThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace atf
