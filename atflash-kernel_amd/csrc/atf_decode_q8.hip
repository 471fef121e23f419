// Windowed split-KV decode over the paged cache of 8-bit floats: decode_kernel's
// attention with half its bytes.
//
// Mathematics.  A page's keys are K = code 2^eK and its values V = code 2^eV (e4m3
// codes, one exponent per page, kv head and half).  S = scale q K^T, O = softmax(S) V on
// bf16 matrix instructions: e4m3 has 4 significant bits and the scales are powers of
// two, so code 2^e is a bf16 number exactly (v_cvt_scalef32_pk_bf16_fp8: two codes times
// the scale an instruction).  Q (rotated in fp32) and P would lose bits as bf16, and so
// are split in two: x = hi + lo, hi = bf16(x), lo = bf16(x - hi), 2^-17 of x left.  With
// up to 8 query heads a kv head (kWide false) this costs no matrix instruction: columns
// 0-7 of an MFMA hold the hi parts of the heads and columns 8-15 their lo parts, of Q
// and of P alike, and the two halves of the result are added (S: a row rotation of the
// lanes; O: once, at the end).  Larger groups take every MFMA twice.  The running
// maximum, the sum and O are fp32; the output is rounded once.
//   Error against 64 bits (2-norm): 1.7e-3, bf16's own; with Q and P rounded to bf16
// it was 2.8e-3 to 4.3e-3.
//
// Layout (atf_common.h): a page's block is 4 KB, V and then K, in the order in which
// the lanes of a wave take them: four loads of 16 bytes a lane, each 1 KB of
// consecutive bytes, bring in a whole page.
//   K: load j, lane (token t = lane % 16, g = lane / 16): the two slices of level
//      4j + g.  Slice i of it is the lane's share of MFMA 2j + i, whose 32 dims are
//      slice i of levels 4j .. 4j + 3.
//   V: load j, lane (row r, g): dims 8r + 4j .. + 3 of tokens 4g .. 4g + 3; dim d of them,
//      of two pages, is the lane's share of MFMA 4j + d, whose row r is dim 8r + 4j + d.
// The window shortens the K read to whole levels (256 bytes); a last odd slice is
// zeroed in registers with the per-key rule's.
//
// Work.  A sequence of P pages is cut into ceil(P / C) splits (C: a.pages_per_split, from
// the call's sizes), page s, s + n, s + 2n, ... to split s of n; a workgroup of 8 or 12
// waves takes a split of a kv head, each wave two pages at a time.  So the splits of a
// ragged batch are all about C pages, long sequences have more of them, and a sequence's
// results do not depend on the lengths of others.
//
// What bounds it.  The bytes of the pages: each is read once.  1 x 131072 tokens (28 / 4
// heads, window OFF, 134 MB): 29.2 us a call with the merge, 4.6 TB/s; 40 x 8192 under the
// level rule 57.8 us, 4.9 TB/s, where a large copy reaches 4.7.  A stream of the same 134 MB
// in 4 KB blocks without any arithmetic takes 20.8 us: the difference is the start (length,
// table entry, page: three round trips one behind the other), the combination of the
// waves at the end, and the merge (4 us).  At 40 x 8192 the vector units are busy for 28%
// of the time and a wave waits for memory for 63% of its own; more pairs of pages in
// flight a wave were not better, they take the registers of other waves.
#include "atf_decode_common.h"

namespace atf {

// Waves of a workgroup: 8, two workgroups to a CU; 12 where every workgroup has a CU of
// its own and its splits are long.  kQFirst: the rows of Q and their (cos, sin) are
// requested ahead of the first pages (loads return in order) and made ready while those
// are on their way.  Measured, us a call with 8 waves, 8 and Q first, 12 and Q first (28 / 4
// heads, vec8 k = 2, where nothing else is said):
//   one round, pages a split  16  1 x 8192 (24 / 8)     11.7  11.0  11.4
//                             24  1 x 24576             14.3  13.5  14.3
//                             32  1 x 32768             15.3  14.8  14.7
//                             48  1 x 49152             17.4  17.3  16.4
//                            128  1 x 131072            28.3  29.6  25.9; OFF 30.1  29.8  29.2
//                            128  4 x 16384 (24 / 8)    27.7  28.8  24.9
//                            282  30 of 300 to 9000     38.9  43.7  32.9
//   more rounds                   12 of 1084 to 32768   36.6  39.0  45.8
//                                 40 x 8192, level rule 59.8  59.4  63.4
//                                 64 of 140 to 4096     45.1  46.9  44.9
//   kWide                         1 x 8192 (32 / 2)     12.9  12.3  13.6
//                                 4 x 65536 (32 / 2)    28.3  28.3  27.6
constexpr int kQ8Waves = 8;
constexpr int kQ8WavesLong = 12;
constexpr int kQ8LongPages = 32;  // of a split, from which on 12 waves take it

// A page's block as a range-checked buffer: V, then the first ns slices of K (whole levels);
// empty for a page past the sequence or an entry outside the pool.  What lies past the
// range is zero without a memory request.
struct Q8Page {
  __amdgpu_buffer_rsrc_t block;
  uint32_t exps;  // byte offset of the page's two exponents (past the buffer: none, read as 0)
};
__device__ __forceinline__ Q8Page q8_page(const DecHot& hot, int h, int raw, bool in_seq, int ns) {
  const int pg = __builtin_amdgcn_readfirstlane(raw);
  const bool ok = in_seq && static_cast<uint32_t>(pg) < static_cast<uint32_t>(hot.num_pages);
  const uint32_t blk = ok ? static_cast<uint32_t>(pg) * hot.hkv + h : 0u;  // (below 2^31)
  const uint8_t* base = reinterpret_cast<const uint8_t*>(hot.kv_cache) + static_cast<uint64_t>(blk) * kQ8BlockBytes;
  const int range = __builtin_amdgcn_readfirstlane(ok ? kQ8HalfBytes + (ns + 1) / 2 * (kPage * 2 * kSliceDims) : 0);
  return Q8Page{__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, range, kBufferWord3), ok ? 2 * blk : ~0u};
}
__device__ __forceinline__ void q8_load(const __amdgpu_buffer_rsrc_t& block, int lane, int at, u32x4 (&x)[2]) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
    x[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                         block, (static_cast<uint32_t>(lane) << 4) + at + j * 1024u, 0, kLoadStream));
}
__device__ __forceinline__ uint32_t q8_exps(const __amdgpu_buffer_rsrc_t& all, const Q8Page& p) {
  return static_cast<uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(all, p.exps, 0, 0));  // eV | eK << 8
}

// 2^e as a float, e the signed byte at bit kAt of w (the cache's exponents are normal floats).
template <int kAt>
__device__ __forceinline__ float q8_scale(uint32_t w) {
  const int e = static_cast<int>(w << (24 - kAt)) >> 24;
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
// Four codes times 2^e as bf16.
__device__ __forceinline__ u32x2 q8_bf16(uint32_t codes, float scale) {
  return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true))};
}
__device__ __forceinline__ bf16x8 join(const u32x2& lo, const u32x2& hi) {
  return __builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], hi[0], hi[1]});
}

// Two values less `m` times their bf16 parts (m = 0: as they are), as bf16.
__device__ __forceinline__ uint32_t pack_part(float x, float y, float m) {
  const uint32_t w = pack_bf16x2(x, y);
  return pack_bf16x2(__builtin_fmaf(-m, __uint_as_float(w << 16), x), __builtin_fmaf(-m, __uint_as_float(w & 0xffff0000u), y));
}

// The slices a page reads, counted by lane (zc: page_slices; the level rule's table holds
// each level's entry for its two slices, and level 0 has no limit), and whether some of
// them are to be zeroed by key: a boundary inside the page, or a last level of which
// only the first slice is read.
template <bool kPerKey>
__device__ __forceinline__ void q8_slices(int zc, int p, int N, int& ns, bool& mask) {
  const int z_young = (N - 1) - (p * kPage + kPage - 1);
  if constexpr (kPerKey) {
    const int cy = __builtin_popcountll(__builtin_amdgcn_ballot_w64(zc >= z_young));
    const int co = __builtin_popcountll(__builtin_amdgcn_ballot_w64(zc >= z_young + kPage - 1));
    ns = cy;
    mask = co != cy || (cy & 1) != 0;
  } else {
    ns = __builtin_popcountll(__builtin_amdgcn_ballot_w64(zc >= max(z_young, 0)));
    mask = false;
  }
}

// Splits of a sequence of `pages` pages.
__device__ __forceinline__ int q8_splits(int pages, int pages_per_split, int n_splits) {
  return n_splits == 1 ? 1 : max(1, (pages + pages_per_split - 1) / pages_per_split);
}

template <bool kPerKey, bool kWide, int kWaves, bool kQFirst>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(kWaves == kQ8WavesLong ? 3 : kWide ? 2 : 4)))
void decode_q8_kernel(const int32_t* page_table, const int32_t* seq_lens, const uint16_t* kv_cache, int max_pages,
                      int pages_per_split, int max_seq_len, int hkv, int num_pages, int n_splits, DecodeArgs a) {
  const DecHot hot{page_table, seq_lens, kv_cache, max_pages, pages_per_split, max_seq_len, hkv, num_pages, n_splits};
  // wave partials
  __shared__ __attribute__((aligned(16))) float sh_o[kWaves * kDecMaxGroup * kD];
  __shared__ float sh_m[kWaves * kDecMaxGroup], sh_l[kWaves * kDecMaxGroup];
  // The splits are turned by head and sequence: workgroups go to the XCDs in turn, and
  // without this the sequences that have few splits would all lie on the first ones (12
  // sequences of 1084 to 32768 tokens, 24 / 8 heads, vec8 k = 2: 66.5 us a call).
  const int h = blockIdx.y, b = blockIdx.z, s = (blockIdx.x + h + b) % n_splits;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, t = lane & 15, g = lane >> 4;
  const float NEG_INF = -__builtin_huge_valf();
  const float c = a.scale_log2;
  // Pair i of this wave is pages p and p + n, p = s + 2 n (wave + kWaves i).  The entries of the
  // first two pairs are fetched together with the length, as if the sequence had the
  // call's longest length (a round trip less where it has as many splits).
  const int32_t* row = page_table + static_cast<int64_t>(b) * max_pages;
  int ent[2], ent_next[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    ent[u] = row[min(s + n_splits * (2 * wave + u), max_pages - 1)];
    ent_next[u] = row[min(s + n_splits * (2 * (wave + kWaves) + u), max_pages - 1)];
  }
  // Q^T fragments: fragment m is slice 2g + m % 2 + 8 (m / 2) of a head.  Lane t holds head
  // t % 8, its hi part for t < 8, its lo part above; kWide: head t, both parts.
  const int head = kWide ? t : t & 7;
  u32x4 x[4];
  float cs[4][8];
  auto request_q = [&] {
    const uint16_t* qrow = a.q + static_cast<int64_t>(b) * a.q_sb +
                           static_cast<int64_t>(h * a.group + min(head, a.group - 1)) * a.q_sh;
    if (a.layout == kLayoutHalfSplit) {
#pragma unroll
      for (int m = 0; m < 4; ++m) x[m] = load_slice(qrow, kLayoutHalfSplit, 2 * g + (m & 1) + 8 * (m >> 1));
    } else {
#pragma unroll
      for (int m = 0; m < 4; ++m) x[m] = load_slice(qrow, kLayoutSortedPair, 2 * g + (m & 1) + 8 * (m >> 1));
    }
  };
  auto request_cs = [&](int pos) {
    if (a.rope_cs != nullptr) {
#pragma unroll
      for (int m = 0; m < 4; ++m) load_cs4(a.rope_cs, pos, slice_pair0(2 * g + (m & 1) + 8 * (m >> 1)), cs[m]);
    }
  };
  if constexpr (kQFirst) request_q();
  const int N = max(0, min(seq_lens[b], max_seq_len));
  const int n_pages = (N + kPage - 1) / kPage;
  const int n = q8_splits(n_pages, pages_per_split, n_splits);
  if (s >= n) return;
  if constexpr (kQFirst) request_cs(max(N - 1, 0));
  const int step = 2 * kWaves * n;
  int p = s + 2 * n * wave;
  auto fetch = [&](int page) { return row[max(min(page, n_pages - 1), 0)]; };
  if (n != n_splits) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      ent[u] = fetch(p + u * n);
      ent_next[u] = fetch(p + step + u * n);
    }
  }
  int zc = INT32_MIN;  // lane s < 16: zhi8[s], the others a limit that no age meets
#pragma unroll
  for (int i = 0; i < kSlices; ++i)
    if (lane == i) zc = !kPerKey && i < 2 ? INT32_MAX : a.st.zhi[i];
  const __amdgpu_buffer_rsrc_t all_exps =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.kv_exps), 0, 2 * num_pages * hkv, kBufferWord3);

  // Entries of the next pair lie in `ent` when a pair is worked on; those of the one
  // behind it are requested before the next pair's loads.
  u32x4 K[2][2], V[2][2];
  uint32_t e[2];
  bool mask[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    int ns;
    q8_slices<kPerKey>(zc, p + u * n, N, ns, mask[u]);
    const Q8Page page = q8_page(hot, h, ent[u], p + u * n < n_pages, ns);
    e[u] = q8_exps(all_exps, page);
    q8_load(page.block, lane, kQ8HalfBytes, K[u]);
    q8_load(page.block, lane, 0, V[u]);
    ent[u] = ent_next[u];
  }

  if constexpr (!kQFirst) {
    request_q();
    request_cs(max(N - 1, 0));
  }
  u32x4 Qf[4], Ql[kWide ? 4 : 1];
  {
    const bool valid = head < a.group && N > 0;
    const float part = !kWide && t >= 8 ? 1.f : 0.f;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      float v[8], y[8];
      unpack8(x[m], v);
      if (a.rope_cs != nullptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] = rope_first(v[i], v[4 + i], cs[m][2 * i], cs[m][2 * i + 1]);
          y[4 + i] = rope_second(v[i], v[4 + i], cs[m][2 * i], cs[m][2 * i + 1]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = v[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        Qf[m][i] = valid ? pack_part(y[2 * i], y[2 * i + 1], part) : 0u;
        if constexpr (kWide) Ql[m][i] = valid ? pack_part(y[2 * i], y[2 * i + 1], 1.f) : 0u;
      }
    }
  }
  // per-key rule: the distance limits of the lane's slices
  int zl[4] = {0, 0, 0, 0};
#pragma unroll
  for (int m = 0; m < 4 && kPerKey; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (g == i) zl[m] = a.st.zhi[2 * i + (m & 1) + 8 * (m >> 1)];
  const float p_part = !kWide && t >= 8 ? 1.f : 0.f;

  f32x4 O[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) O[e] = f32x4{};
  float m_run = NEG_INF, l_run = 0.f;

  float msc = 0.f;   // m_run in log2 units
  bool first = true;
  for (; p < n_pages; p += step) {
#pragma unroll
    for (int u = 0; u < 2; ++u) ent_next[u] = fetch(p + 2 * step + u * n);
    f32x4 S[2];
    float sv[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (kPerKey && mask[u]) {
        const int age = (N - 1) - ((p + u * n) * kPage + t);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          if (age > zl[m]) {
            K[u][m >> 1][2 * (m & 1)] = 0u;
            K[u][m >> 1][2 * (m & 1) + 1] = 0u;
          }
      }
      const float sk = q8_scale<8>(e[u]);
      sv[u] = q8_scale<0>(e[u]);
      S[u] = f32x4{};
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const bf16x8 A = join(q8_bf16(K[u][m >> 1][2 * (m & 1)], sk), q8_bf16(K[u][m >> 1][2 * (m & 1) + 1], sk));
        S[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, __builtin_bit_cast(bf16x8, Qf[m]), S[u], 0, 0, 0);
        if constexpr (kWide) S[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, __builtin_bit_cast(bf16x8, Ql[m]), S[u], 0, 0, 0);
      }
    }
    // K of the next pair (past the sequence: nothing)
    Q8Page next[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int q = p + step + u * n;
      int ns;
      q8_slices<kPerKey>(zc, q, N, ns, mask[u]);
      next[u] = q8_page(hot, h, ent[u], q < n_pages, ns);
      e[u] = q8_exps(all_exps, next[u]);
      q8_load(next[u].block, lane, kQ8HalfBytes, K[u]);
    }
    // S lane layout: query head t (hi part; lo part in t + 8), tokens 4g + i
    if constexpr (!kWide) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) S[u][i] += row_ror<8>(S[u][i]);
    }
    if ((p + n + 1) * kPage > N) {  // the sequence ends in this pair, or between its pages
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int left = N - (p + u * n) * kPage - 4 * g;  // of the lane's four tokens
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i >= left) S[u][i] = NEG_INF;
        // V codes past the sequence to zero, so that 0 * V stays 0
        const uint32_t keep = left >= 4 ? 0xffffffffu : (1u << (8 * max(left, 0))) - 1u;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int w = 0; w < 4; ++w) V[u][j][w] &= keep;
      }
    }
    // P against the reference maximum so far.  It moves only where a lane's P add up to
    // more than 256 (a score above it by 5 or more), and with the first pair.
    float P[2][4];
    auto exps = [&] {
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          P[u][i] = fast_exp2(__builtin_fmaf(S[u][i], c, -msc));
          sum += P[u][i];
        }
      return sum;
    };
    float sum = exps();
    if (__builtin_amdgcn_ballot_w64(first || !(sum <= 256.f)) != 0) {
      float mx = fmaxf(fmaxf(fmaxf(S[0][0], S[0][1]), fmaxf(S[0][2], S[0][3])),
                       fmaxf(fmaxf(S[1][0], S[1][1]), fmaxf(S[1][2], S[1][3])));
      mx = quad_max(mx);
      if (mx > m_run) {
        const float alpha = m_run == NEG_INF ? 0.f : fast_exp2((m_run - mx) * c);
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < 8; ++d) O[d] *= alpha;
        m_run = mx;
        msc = mx * c;
      }
      first = false;
      sum = exps();
    }
    l_run += sum;
    u32x2 Ph[2], Pl[kWide ? 2 : 1];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      Ph[u] = u32x2{pack_part(P[u][0], P[u][1], p_part), pack_part(P[u][2], P[u][3], p_part)};
      if constexpr (kWide) Pl[u] = u32x2{pack_part(P[u][0], P[u][1], 1.f), pack_part(P[u][2], P[u][3], 1.f)};
    }
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const bf16x8 A = join(q8_bf16(V[0][d >> 2][d & 3], sv[0]), q8_bf16(V[1][d >> 2][d & 3], sv[1]));
      O[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, join(Ph[0], Ph[1]), O[d], 0, 0, 0);
      if constexpr (kWide) O[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, join(Pl[0], Pl[1]), O[d], 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      q8_load(next[u].block, lane, 0, V[u]);
      ent[u] = ent_next[u];
    }
  }

  // ---- the split's partial: combine the wave partials in LDS ----
  const float l_tot = quad_sum(l_run);
  if constexpr (!kWide) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) O[e][i] += row_ror<8>(O[e][i]);
  }
  if (t < a.group) {
    // O[e][i]: dim 8 (4g + i) + e
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float* o = &sh_o[(wave * kDecMaxGroup + t) * kD + 8 * (4 * g + i)];
      *reinterpret_cast<f32x4*>(o) = f32x4{O[0][i], O[1][i], O[2][i], O[3][i]};
      *reinterpret_cast<f32x4*>(o + 4) = f32x4{O[4][i], O[5][i], O[6][i], O[7][i]};
    }
    if (lane < 16) {
      sh_m[wave * kDecMaxGroup + t] = m_run;
      sh_l[wave * kDecMaxGroup + t] = l_tot;
    }
  }
  __syncthreads();
  store_split<kWaves>(a, (static_cast<int64_t>(b) * hkv + h) * n_splits + s, n == 1, h, b, sh_o, sh_m, sh_l);
}

// The merge of the splits that each sequence has (those with one have written their output).
__global__ __launch_bounds__(512) void decode_q8_merge_kernel(const int32_t* seq_lens, int pages_per_split, int max_seq_len,
                                                              MergeArgs a) {
  const int N = max(0, min(seq_lens[blockIdx.z], max_seq_len));
  const int n = q8_splits((N + kPage - 1) / kPage, pages_per_split, a.n_splits);
  if (n > 1) merge_splits<false>(a, n);
}

// The same where a sequence has kMost splits at most: a thread takes 4 dims of a query
// head and asks for all of their partials at once, so that no lanes wait for splits that
// are not there.  Measured, us a call with decode_q8_merge_kernel and with this one: 3
// splits 40 x 8192 59.3, 56.1; 4 1 x 1003 10.5, 9.6; 5 20 of 200 to 3000 (32 / 2 heads)
// 14.3, 13.5; 8 4 x 16384 (24 / 8) 24.8, 24.6; 16 1 x 4096 10.8, 12.6, 12 of 1084 to 32768
// 36.6, 37.9: up to 8 splits.
constexpr int kMergeFewThreads = 256;
template <int kMost>
__global__ __launch_bounds__(kMergeFewThreads) void decode_q8_merge_few_kernel(const int32_t* seq_lens, int pages_per_split,
                                                                  int max_seq_len, MergeArgs a, int rows) {
  const int at = blockIdx.x * kMergeFewThreads + threadIdx.x;
  const int row = at / (kD / 4), md4 = 4 * (at % (kD / 4));
  if (row >= rows) return;
  const int pair = row / a.group, mg = row - pair * a.group;  // (sequence, kv head), query head of it
  const int b = pair / a.hkv;
  const int64_t part = static_cast<int64_t>(pair) * a.n_splits * kDecMaxGroup + mg;
  f32x2 ml[kMost];
  f32x4 o[kMost];
  const int N = max(0, min(seq_lens[b], max_seq_len));
  const int n = q8_splits((N + kPage - 1) / kPage, pages_per_split, a.n_splits);
  if (n <= 1) return;
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    const int64_t i = part + static_cast<int64_t>(min(j, n - 1)) * kDecMaxGroup;
    ml[j] = *reinterpret_cast<const f32x2*>(a.ws_ml + 2 * i);
    o[j] = *reinterpret_cast<const f32x4*>(a.ws_o + i * kD + md4);
  }
  float top = ml[0][0];
#pragma unroll
  for (int j = 1; j < kMost; ++j) top = fmaxf(top, ml[j][0]);
  float L = 0.f;
  f32x4 acc = f32x4{};
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    const float w = j < n && ml[j][0] != -__builtin_huge_valf() ? fast_exp2((ml[j][0] - top) * a.scale_log2) : 0.f;
    L += w * ml[j][1];
    acc += w * o[j];
  }
  store_merged(a, b, (pair - b * a.hkv) * a.group + mg, md4, L, acc);
}

hipError_t launch_decode_q8(const DecodeArgs& a, hipStream_t s) {
  if (a.batch <= 0) return hipSuccess;
  const dim3 grid(a.n_splits, a.hkv, a.batch);
#define ATF_Q8_LAUNCH(PK, WIDE, W, QF)                                                                                  \
  hipLaunchKernelGGL((decode_q8_kernel<PK, WIDE, W, QF>), grid, dim3((W) * 64), 0, s, a.page_table, a.seq_lens,          \
                     a.kv_cache, a.max_pages, a.pages_per_split, a.max_seq_len, a.hkv, a.num_pages, a.n_splits, a)
  const bool one_round = static_cast<int64_t>(a.n_splits) * a.hkv * a.batch <= 256;
  if (a.group > 8) {
    if (a.per_key) ATF_Q8_LAUNCH(true, true, kQ8Waves, true); else ATF_Q8_LAUNCH(false, true, kQ8Waves, true);
  } else if (!one_round) {
    if (a.per_key) ATF_Q8_LAUNCH(true, false, kQ8Waves, false); else ATF_Q8_LAUNCH(false, false, kQ8Waves, false);
  } else if (a.pages_per_split >= kQ8LongPages) {
    if (a.per_key) ATF_Q8_LAUNCH(true, false, kQ8WavesLong, true); else ATF_Q8_LAUNCH(false, false, kQ8WavesLong, true);
  } else {
    if (a.per_key) ATF_Q8_LAUNCH(true, false, kQ8Waves, true); else ATF_Q8_LAUNCH(false, false, kQ8Waves, true);
  }
#undef ATF_Q8_LAUNCH
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  if (a.n_splits > 1) {
    const MergeArgs m{a.ws_ml, a.ws_o, a.out, a.o_sb, a.o_sh, a.n_splits, a.group, a.hkv, a.scale_log2};
    const int64_t rows = static_cast<int64_t>(a.batch) * a.hkv * a.group;
    if (a.n_splits <= 8 && rows <= INT32_MAX / (kD / 4))
      hipLaunchKernelGGL(a.n_splits <= 4 ? decode_q8_merge_few_kernel<4> : decode_q8_merge_few_kernel<8>,
                         dim3((rows * (kD / 4) + kMergeFewThreads - 1) / kMergeFewThreads), dim3(kMergeFewThreads), 0, s,
                         a.seq_lens, a.pages_per_split, a.max_seq_len, m, static_cast<int>(rows));
    else
      hipLaunchKernelGGL(decode_q8_merge_kernel, dim3(kMergeChunks, a.hkv, a.batch), dim3(512), 0, s, a.seq_lens,
                         a.pages_per_split, a.max_seq_len, m);
    return hipGetLastError();
  }
  return hipSuccess;
}

}  // namespace atf
