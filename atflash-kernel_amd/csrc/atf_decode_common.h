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
// part: the partial's index in the workspace; whole: the split is the whole sequence.
template <int kWaves>
__device__ __forceinline__ void store_split(const DecodeArgs& a, int64_t part, bool whole, int h, int b,
                                            const float* sh_o, const float* sh_m, const float* sh_l) {
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
    if (whole) {  // write the output
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

// Log-sum-exp merge of the split partials, launched after decode_kernel when
// n_splits > 1.  One workgroup per (16-dim chunk, kv head, sequence), so that
// the merge's loads spread over 8 CUs per (sequence, kv head) (4 chunks of 32
// dims were 0.6-0.75 us slower per call, 16 chunks of 8 dims 0.2 us).  Thread
// t takes 4 dims of its chunk and, for query head mg, every H-th split
// starting at hh (H = 16 for G <= 8, 8 for larger groups).  It loads the
// (m, l) and o of up to kMergeBatch splits before using any of them, so with
// up to 64 splits (32 for G > 8) the merge costs one memory round trip; more
// splits are folded in batch by batch with a running max.  The H partial
// merges of a (head, dims) sit in lanes 4k + (t % 4) of one wave (half wave
// for G > 8) and are combined by DPP row rotations and permlane swaps, VALU
// moves without LDS or a workgroup barrier.
constexpr int kMergeChunks = 8;
constexpr int kMergeDims = kD / kMergeChunks;          // dims per workgroup
constexpr int kMergeLanes = kMergeDims / 4;            // lanes per (head, split group), 4 dims each
constexpr int kMergeRowsPerWave = 64 / kMergeLanes;    // (head, split group) rows per wave
constexpr int kMergeBatch = 4;                         // splits loaded per thread before use
static_assert(kMergeChunks * kMergeDims == kD && kMergeLanes == 4 && kDecMaxGroup <= 16,
              "merge layout: 4 lanes per (head, split group), one or two heads per wave (8 waves: 8 heads for "
              "G <= 8, 16 for larger groups)");

// The merge kernel's arguments are scalars (14 dwords), preloaded into SGPRs
// with the dispatch, so the partial loads are issued at once instead of after
// a read of an argument block.
struct MergeArgs {
  const float* ws_ml;
  const float* ws_o;
  uint16_t* out;
  int64_t o_sb, o_sh;
  int n_splits, group, hkv;
  float scale_log2;
};

// Two (m, l, o) partials merged by log-sum-exp.
__device__ __forceinline__ void merge_pair(float& m, float& l, f32x4& o, float mp, float lp, const f32x4& op,
                                           float c) {
  const float NEG_INF = -__builtin_huge_valf();
  const float M = fmaxf(m, mp);
  if (M != NEG_INF) {
    const float w = fast_exp2((m - M) * c), wp = fast_exp2((mp - M) * c);  // an empty side: m = -inf -> 0
    l = w * l + wp * lp;
    o = w * o + wp * op;
    m = M;
  }
}

// Lane (l + n) % 16 of l's 16-lane row (DPP row rotation: a VALU move, no LDS).
template <int kN>
__device__ __forceinline__ float row_ror(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + kN, 0xF, 0xF, false));
}

// The partial of lane l merged with those of lanes l + 4, l + 8, l + 12 of its
// row (two row rotations), then with the rows l ^ 16 (and l ^ 32 when
// `whole_wave`) by the gfx950 permlane swaps, which hand each lane the value of
// the lane one row (two rows) away: afterwards every lane of a group {4h + q}
// holds the merge of the group's partials.  Every lane takes part; the caller
// keeps control flow uniform around it.
// merge_rows: the row rotations alone, for groups that lie in a 16-lane row.
__device__ __forceinline__ void merge_rows(float& m, float& l, f32x4& o, float c) {
  {
    f32x4 op;
#pragma unroll
    for (int i = 0; i < 4; ++i) op[i] = row_ror<8>(o[i]);
    merge_pair(m, l, o, row_ror<8>(m), row_ror<8>(l), op, c);
  }
  {
    f32x4 op;
#pragma unroll
    for (int i = 0; i < 4; ++i) op[i] = row_ror<4>(o[i]);
    merge_pair(m, l, o, row_ror<4>(m), row_ror<4>(l), op, c);
  }
}
__device__ __forceinline__ void merge_lane_groups(float& m, float& l, f32x4& o, bool whole_wave, float c) {
  merge_rows(m, l, o, c);
  // a swap of a register with itself: result [0] holds rows (0, 0, 2, 2) and
  // result [1] rows (1, 1, 3, 3) of the value (32-lane swap: halves (0, 0) and
  // (1, 1)), so merging [0] with [1] merges each lane with its partner lane
  auto swap16 = [](float x) {
    return __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  };
  auto swap32 = [](float x) {
    return __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  };
  {
    const auto sm = swap16(m), sl = swap16(l);
    f32x4 o0, o1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto so = swap16(o[i]);
      o0[i] = __uint_as_float(so[0]);
      o1[i] = __uint_as_float(so[1]);
    }
    m = __uint_as_float(sm[0]);
    l = __uint_as_float(sl[0]);
    o = o0;
    merge_pair(m, l, o, __uint_as_float(sm[1]), __uint_as_float(sl[1]), o1, c);
  }
  if (whole_wave) {  // uniform over the launch
    const auto sm = swap32(m), sl = swap32(l);
    f32x4 o0, o1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto so = swap32(o[i]);
      o0[i] = __uint_as_float(so[0]);
      o1[i] = __uint_as_float(so[1]);
    }
    m = __uint_as_float(sm[0]);
    l = __uint_as_float(sl[0]);
    o = o0;
    merge_pair(m, l, o, __uint_as_float(sm[1]), __uint_as_float(sl[1]), o1, c);
  }
}

// The output row of query head hq_idx, dims md4 .. +3.
__device__ __forceinline__ void store_merged(const MergeArgs& a, int b, int hq_idx, int md4, float l, const f32x4& o) {
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint16_t* out = a.out + static_cast<int64_t>(b) * a.o_sb + static_cast<int64_t>(hq_idx) * a.o_sh + md4;
  u32x2 pk;
  pk[0] = pack_bf16x2(o[0] * inv, o[1] * inv);
  pk[1] = pack_bf16x2(o[2] * inv, o[3] * inv);
  *reinterpret_cast<u32x2*>(out) = pk;
}

// The wave partials of a split (decode_wave_kernel's; split: its index in the call)
// combined, for query head mg of the group and dims md4 .. +3.
__device__ __forceinline__ void load_wave_split(const MergeArgs& a, int64_t split, int mg, int md4, float& M, float& L,
                                                f32x4& acc) {
  combine_waves<kDecWaves>(
      [&](int w, float& m, float& l, f32x4& o) {
        const int64_t u = split * kDecWaves + w;
        const float* ml = a.ws_ml + u * 2 * a.group + mg;
        m = ml[0];
        l = ml[a.group];
        o = *reinterpret_cast<const f32x4*>(a.ws_o + (u * a.group + mg) * kD + md4);
      },
      a.scale_log2, M, L, acc);
}

// kWavePartials: the partials are decode_wave_kernel's, a split's combined as it is loaded.
// count: the splits that hold the pair's partials, of the n_splits it has room for.
template <bool kWavePartials>
__device__ __forceinline__ void merge_splits(const MergeArgs& a, int count) {
  const int chunk = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int64_t part0 = (static_cast<int64_t>(b) * a.hkv + h) * a.n_splits;  // split 0's partial
  const int tid = threadIdx.x;
  const float NEG_INF = -__builtin_huge_valf();
  const float c = a.scale_log2;
  const int H = (a.group <= 8) ? kMergeRowsPerWave : kMergeRowsPerWave / 2;
  const int row = tid / kMergeLanes;  // (head, split group)
  const int mg = row / H, hh = row - (row / H) * H;
  const int q4 = 4 * (tid % kMergeLanes);
  const int md4 = chunk * kMergeDims + q4;
  const bool mact = mg < a.group;
  float m_t = NEG_INF, L_t = 0.f;
  f32x4 acc_t = f32x4{};
  if (mact) {
    for (int j0 = hh; j0 < count; j0 += kMergeBatch * H) {
      f32x2 mlv[kMergeBatch];
      f32x4 ov[kMergeBatch];
#pragma unroll
      for (int j = 0; j < kMergeBatch; ++j) {
        const int sp = j0 + j * H;
        mlv[j] = f32x2{NEG_INF, 0.f};
        ov[j] = f32x4{};
        if (sp < count) {
          if constexpr (kWavePartials) {
            float M, L;
            load_wave_split(a, part0 + sp, mg, md4, M, L, ov[j]);
            mlv[j] = f32x2{M, L};
          } else {
            const int64_t pi = (part0 + sp) * kDecMaxGroup + mg;
            mlv[j] = *reinterpret_cast<const f32x2*>(a.ws_ml + pi * 2);
            ov[j] = *reinterpret_cast<const f32x4*>(a.ws_o + pi * kD + md4);
          }
        }
      }
      float mb = m_t;
#pragma unroll
      for (int j = 0; j < kMergeBatch; ++j) mb = fmaxf(mb, mlv[j][0]);
      if (mb != NEG_INF) {
        const float r = fast_exp2((m_t - mb) * c);  // m_t = -inf -> 0
        L_t *= r;
        acc_t *= r;
#pragma unroll
        for (int j = 0; j < kMergeBatch; ++j) {
          const float wt = fast_exp2((mlv[j][0] - mb) * c);  // empty split: m = -inf -> 0
          L_t += wt * mlv[j][1];
          acc_t += wt * ov[j];
        }
        m_t = mb;
      }
    }
  }
  // every lane of the wave takes part in the exchanges (inactive rows hold an
  // empty partial); lanes 4k + (t % 4), k < H, hold one (head, dims): 16
  // groups per wave for G <= 8, 8 per half wave above
  merge_lane_groups(m_t, L_t, acc_t, H == 16, c);
  if (mact && hh == 0) store_merged(a, b, h * a.group + mg, md4, L_t, acc_t);
}

}  // namespace atf
