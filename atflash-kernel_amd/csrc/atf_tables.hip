// Block tables and slot maps from request lengths, on the GPU.
//
// A sequence of L tokens that gets n more needs the pages ceil(L / 16) ..
// ceil((L + n) / 16) - 1.  They are taken from the end of the free pages, sequence by
// sequence, as PagedKVCache.reserve takes them on the host: the r-th page of a call
// is free[count - 1 - r].  Token t of the call, the i-th new one of sequence b, is at
// position p = L_b + i and in slot 16 page(p / 16) + p % 16.
//   Latency bound: 8 bytes a sequence read and 8 written, 4 a page each way, 12 a token
// written; 64 sequences with a token each
// 3.5 us, 300 with 75000 tokens 5.6 us (1.5 MB).  One launch: every workgroup
// forms the prefix sums of all sequences itself (tokens and pages, in LDS) instead of
// waiting for one that does, and nothing it reads is written by another (new pages are
// entered behind the columns that are read; lengths and the free count come out as new
// arrays).
#include "atf_launch.h"

namespace atf {

constexpr int kTabThreads = 256;

// The last i with at[i] <= x, at[0] = 0 <= x < at[n], at not decreasing.
__device__ __forceinline__ int last_at_most(const int32_t* at, int n, int x) {
  int lo = 0, hi = n;  // at[lo] <= x < at[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(int64_t tokens) { return static_cast<int>((tokens + kPage - 1) / kPage); }

__global__ __launch_bounds__(kTabThreads) void extend_tables_kernel(ExtendTablesArgs a) {
  extern __shared__ int32_t sh[];
  int32_t* cu = sh;                   // [batch + 1] first token of each sequence
  int32_t* base = sh + a.batch + 1;   // [batch + 1] first page, of the call's
  __shared__ int32_t part[2][kTabThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto length = [&](int b) { return max(a.seq_lens[b], 0); };
  auto fresh = [&](int b) { return max(a.new_lens[b], 0); };
  int carry_t = 0, carry_p = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kTabThreads) {
    const int b = b0 + tid;
    int n = 0, need = 0;
    if (b < a.batch) {
      const int len = length(b);
      n = fresh(b);
      need = max(min(pages_of(static_cast<int64_t>(len) + n), a.max_pages) - pages_of(len), 0);
      if (blockIdx.x == 0)
        a.lens_out[b] = static_cast<int>(min(static_cast<int64_t>(len) + n, static_cast<int64_t>(INT32_MAX)));
    }
    int st = n, sp = need;  // inclusive sums of the wave, then of the workgroup
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int ut = __shfl_up(st, m), up = __shfl_up(sp, m);
      st += lane >= m ? ut : 0;
      sp += lane >= m ? up : 0;
    }
    if (lane == 63) {
      part[0][wave] = st;
      part[1][wave] = sp;
    }
    __syncthreads();
    int all_t = 0, all_p = 0;
#pragma unroll
    for (int w = 0; w < kTabThreads / 64; ++w) {
      st += w < wave ? part[0][w] : 0;
      sp += w < wave ? part[1][w] : 0;
      all_t += part[0][w];
      all_p += part[1][w];
    }
    if (b < a.batch) {
      cu[b] = carry_t + st - n;
      base[b] = carry_p + sp - need;
    }
    carry_t += all_t;
    carry_p += all_p;
    __syncthreads();
  }
  if (tid == 0) {
    cu[a.batch] = carry_t;
    base[a.batch] = carry_p;
  }
  __syncthreads();
  const int count = a.free_count[0];
  auto page_at = [&](int r) {  // the r-th page of the call; -1 where the free pages ran out
    return r < count && count - 1 - r < a.num_free ? a.free_pages[count - 1 - r] : -1;
  };
  if (blockIdx.x == 0) {
    for (int b = tid; b <= a.batch; b += kTabThreads) a.cu_out[b] = cu[b];
    if (tid == 0) a.free_left[0] = count - carry_p;
  }
  const int at = blockIdx.x * kTabThreads + tid, step = gridDim.x * kTabThreads;
  for (int r = at; r < carry_p; r += step) {
    const int b = last_at_most(base, a.batch, r);
    a.page_table[static_cast<int64_t>(b) * a.max_pages + pages_of(length(b)) + (r - base[b])] = page_at(r);
  }
  for (int t = at; t < a.total; t += step) {
    int pos = -1;
    int64_t slot = -1;
    if (t < carry_t) {
      const int b = last_at_most(cu, a.batch, t);
      const int len = length(b), had = pages_of(len);
      const int64_t at64 = static_cast<int64_t>(len) + t - cu[b];  // (lengths that make no sense: no page)
      pos = static_cast<int>(min(at64, static_cast<int64_t>(INT32_MAX)));
      const int col = pos / kPage;
      int page = -1;
      if (col < a.max_pages)
        page = col < had ? a.page_table[static_cast<int64_t>(b) * a.max_pages + col] : page_at(base[b] + col - had);
      if (page >= 0 && page < a.num_pages) slot = static_cast<int64_t>(page) * kPage + pos % kPage;
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
  }
}

hipError_t launch_extend_tables(const ExtendTablesArgs& a, hipStream_t s) {
  // a token a thread (at most 1024 workgroups): its search and its loads wait for one
  // another (300 sequences, 75000 tokens: 5.5 us; 8.6 with several tokens a thread)
  const int64_t blocks64 = (static_cast<int64_t>(a.total) + kTabThreads) / kTabThreads;
  const int blocks = static_cast<int>(blocks64 < 1024 ? blocks64 : 1024);
  const size_t lds = 2 * (static_cast<size_t>(a.batch) + 1) * sizeof(int32_t);
  hipLaunchKernelGGL(extend_tables_kernel, dim3(blocks), dim3(kTabThreads), lds, s, a);
  return hipGetLastError();
}

// The pages of finished sequences back to the end of the free pages, row by row of
// `rows` and page by page; their table rows become -1, their lengths 0.  Entries that are
// no page (a row that ran out of pages) are not given back, a row that is named twice or
// holds nothing gives nothing.  One workgroup: the place of a page in the free list
// depends on all before it.
__global__ __launch_bounds__(kTabThreads) void release_tables_kernel(ReleaseTablesArgs a) {
  __shared__ int32_t part[kTabThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int count = min(max(a.free_count[0], 0), a.num_free);
  for (int i = 0; i < a.n_rows; ++i) {
    const int b = a.rows[i];
    if (b < 0 || b >= a.batch) continue;  // uniform
    int32_t* row = a.page_table + static_cast<int64_t>(b) * a.max_pages;
    const int pages = min(pages_of(max(a.seq_lens[b], 0)), a.max_pages);
    for (int p0 = 0; p0 < pages; p0 += kTabThreads) {
      const int p = p0 + tid;
      const int pg = p < pages ? row[p] : -1;
      const bool live = pg >= 0 && pg < a.num_pages;
      const uint64_t mask = __builtin_amdgcn_ballot_w64(live);
      if (lane == 0) part[wave] = __builtin_popcountll(mask);
      __syncthreads();
      int before = 0, all = 0;
#pragma unroll
      for (int w = 0; w < kTabThreads / 64; ++w) {
        before += w < wave ? part[w] : 0;
        all += part[w];
      }
      const int at = count + before +
                     __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                               __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0u));
      if (live && at < a.num_free) a.free_pages[at] = pg;
      if (p < pages) row[p] = -1;
      count = min(count + all, a.num_free);
      __syncthreads();
    }
    if (tid == 0) a.seq_lens[b] = 0;
    __syncthreads();  // (drains the store: a row named again reads length 0)
  }
  if (tid == 0) a.free_count[0] = count;
}

hipError_t launch_release_tables(const ReleaseTablesArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(release_tables_kernel, dim3(1), dim3(kTabThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace atf
