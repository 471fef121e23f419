// Device code shared by the decode kernels over bf16 and 8-bit pages: the pages of a
// split and their order, the window's slices of a page, the combination of wave
// partials, the order of a ragged batch.
#pragma once
#include "atf_launch.h"

namespace atf {

// max / sum over the 4 lanes {l, l^16, l^32, l^48} that hold one query head.
__device__ __forceinline__ float quad_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float quad_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Page order of a split: the split's local page j (0 <= j < its page count)
// is page po + pm * j of the sequence.  Splits of at least kDecIlvMinPages
// pages (one 4-page group per wave of an 8-wave workgroup) interleave
// (po = s, pm = n_splits: split s takes pages s, s + n_splits, ...), so that
// the workgroups of a call sweep the sequence from its oldest to its youngest
// page together and each split holds pages of every age.  Shorter splits (the
// 4-wave workgroups of short contexts) take contiguous runs
// (po = s * pages_per_split, pm = 1).  Measured per call against contiguous
// runs for every split (same box, graph-replayed; pools rotated past the
// last-level cache): with a page table in allocation order (the cache's own
// allocators) Qwen 128K OFF -2 to -4%, k=2 -8 to -10% (three runs), Llama 32K
// OFF -2.5 to -8.5%, k=2 -8.5 to -9.5%, Llama 128K OFF -2.5%, k=2 -5.5%,
// Llama 16K OFF -6.5%, k=2 -12%, Qwen 32K -2%; with randomly permuted pages
// +0.3 to +1.3% at those shapes; at 8K with 4-wave workgroups interleaving lost
// up to 4-6%.  po and pm are known before the sequence length is; count is set
// once it is.
constexpr int kDecIlvMinPages = kDecUnroll * kDecWaves;
struct PageOrder {
  int po, pm;
  int count;  // the split's pages for this sequence
};
__device__ __forceinline__ PageOrder page_order(int s, int n_splits, int pages_per_split) {
  const bool ilv = pages_per_split >= kDecIlvMinPages;
  return PageOrder{ilv ? s : s * pages_per_split, ilv ? n_splits : 1, 0};
}
__device__ __forceinline__ void set_page_count(PageOrder& o, int s, int n_splits, int pages_per_split,
                                               int n_pages) {
  o.count = o.pm != 1 ? (n_pages > s ? (n_pages - s + n_splits - 1) / n_splits : 0)
                      : max(0, min(n_pages - o.po, pages_per_split));  // (n_splits 1: the same count)
}

// Page-table entry of local page j (a vector register; every lane holds the
// same value).  The load is unconditional, its index clamped into the split:
// an entry for a page past the split is fetched but never used (its page is
// not loaded), and a split without pages reads entry po, inside the table
// row.  A load guarded by a branch with a default value would make the
// compiler wait for every outstanding load before the register's next use.
// A wave fetches a page's entry one stride ahead of its use, so the page loads
// are issued without waiting for the table.
__device__ __forceinline__ int dec_fetch_entry(const int32_t* row, const PageOrder& o, int j) {
  return row[o.po + o.pm * max(0, min(j, o.count - 1))];
}

// The fields of the call that the first page loads need, passed as leading
// scalar kernel arguments so that they arrive preloaded in SGPRs (kernarg
// preloading): the page-table and sequence-length loads are issued without
// first waiting for the argument block to be read from memory.
struct DecHot {
  const int32_t* page_table;
  const int32_t* seq_lens;
  const uint16_t* kv_cache;
  int max_pages, pages_per_split, max_seq_len, hkv, num_pages, n_splits;
};

// The slices page p reads and whether an older key of it reads fewer.  Page
// rule (level table): 2 L(p) slices, L(p) = levels of the youngest key's age.
// Per-key rule: the youngest key's slices, #{s : zhi8[s] >= age}; a slice
// boundary falls inside the page when the oldest key's count differs.  Lane
// s < 16 holds zhi8[s] (zc; the other lanes a limit no age meets), so each
// count is one vector compare and the popcount of its ballot (the caller keeps
// every lane active): against 16 scalar compares per count, -0.3 to -1.0 us per
// call at 32K-128K (+0.5 us at Llama 32K), and those in turn were 0.4 us per
// call faster at 128K than walking the slice boundaries page by page with a
// loop, whose branches sat in front of every page load.
template <bool kPerKey>
__device__ __forceinline__ void page_slices(const DecodeArgs& a, int zc, int p, int N, int& ns, bool& mask) {
  const int z_young = (N - 1) - (p * kPage + kPage - 1);
  if constexpr (kPerKey) {
    const int z_old = z_young + kPage - 1;
    const int cy = __builtin_popcountll(__builtin_amdgcn_ballot_w64(zc >= z_young));
    const int co = __builtin_popcountll(__builtin_amdgcn_ballot_w64(zc >= z_old));
    ns = cy;
    mask = co != cy;
  } else {
    ns = 2 * levels_of(a.lt, max(0, z_young));
    mask = false;
  }
}

// A split's wave partials (m, l, o) combined by log-sum-exp, wave 0 first: part(w,
// m, l, o) yields wave w's.  An empty split gives (-inf, 0, 0).
template <int kWaves, class Part>
__device__ __forceinline__ void combine_waves(const Part& part, float c, float& M, float& L, f32x4& acc) {
  const float NEG_INF = -__builtin_huge_valf();
  float m[kWaves], l[kWaves];
  f32x4 o[kWaves];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) part(w, m[w], l[w], o[w]);
  M = NEG_INF;
  L = 0.f;
  acc = f32x4{};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) M = fmaxf(M, m[w]);
  if (M != NEG_INF) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float wt = fast_exp2((m[w] - M) * c);  // empty wave: m = -inf -> 0
      L += wt * l[w];
      acc += wt * o[w];
    }
  }
}

// The split's wave partials in LDS combined: the output where the split is the
// whole sequence, otherwise the split's partial for decode_merge_kernel.  Thread t
// owns query heads t / 32 + 2 kWaves j, dims 4 (t % 32) .. +3.
// part: the partial's index in the workspace.
template <int kWaves>
__device__ __forceinline__ void store_split(const DecodeArgs& a, int64_t part, int h, int b, const float* sh_o,
                                            const float* sh_m, const float* sh_l) {
  const float c = a.scale_log2;
  const int tid = threadIdx.x;
  const int d4 = 4 * (tid & 31);
  for (int gq = tid >> 5; gq < a.group; gq += 2 * kWaves) {
    float M, L;
    f32x4 acc;
    combine_waves<kWaves>(
        [&](int w, float& m, float& l, f32x4& o) {
          m = sh_m[w * kDecMaxGroup + gq];
          l = sh_l[w * kDecMaxGroup + gq];
          o = *reinterpret_cast<const f32x4*>(&sh_o[(w * kDecMaxGroup + gq) * kD + d4]);
        },
        c, M, L, acc);
    if (a.n_splits == 1) {  // write the output
      const float inv = L > 0.f ? 1.f / L : 0.f;
      uint16_t* out = a.out + static_cast<int64_t>(b) * a.o_sb + static_cast<int64_t>(h * a.group + gq) * a.o_sh + d4;
      u32x2 pk;
      pk[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
      pk[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<u32x2*>(out) = pk;
    } else {  // the split's partial, merged by decode_merge_kernel
      const int64_t pi = part * kDecMaxGroup + gq;
      *reinterpret_cast<f32x4*>(a.ws_o + pi * kD + d4) = acc;
      if (d4 == 0) *reinterpret_cast<f32x2*>(a.ws_ml + pi * 2) = f32x2{M, L};
    }
  }
}

constexpr int kDecSpreadBatch = 512;  // sequences at most

// The sequence of rank r by length in pages (0: the longest; equal lengths by
// index).  r < batch <= 64 kRegs; every lane of the wave takes part.
template <int kRegs>
__device__ __forceinline__ int nth_longest(const int32_t* seq_lens, int batch, int max_seq_len, int r) {
  const int lane = threadIdx.x & 63;
  int p[kRegs];  // pages of sequence 64 i + lane (-1 past the batch)
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const int b = 64 * i + lane;
    p[i] = b < batch ? (max(0, min(seq_lens[b], max_seq_len)) + kPage - 1) / kPage : -1;
  }
  auto count = [&](int at_least) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kRegs; ++i) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(p[i] >= at_least));
    return n;
  };
  int t = 0;  // the largest page count that more than r sequences reach
  for (int bit = 1 << (31 - __builtin_clz(max_seq_len / kPage + 1)); bit != 0; bit >>= 1)
    if (count(t | bit) > r) t |= bit;
  int k = r - count(t + 1);  // the k-th of the sequences of t pages
  int found = 0;
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const uint64_t eq = __builtin_amdgcn_ballot_w64(p[i] == t);
    const int below = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(eq >> 32),
                                                __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(eq), 0u));
    const uint64_t hit = __builtin_amdgcn_ballot_w64(p[i] == t && below == k);
    if (hit != 0) found = 64 * i + __builtin_ctzll(hit);
    k -= __builtin_popcountll(eq);
  }
  return found;
}

}  // namespace atf
