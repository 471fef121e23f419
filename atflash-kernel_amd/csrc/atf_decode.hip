// Windowed split-KV decode over the paged KV cache (gfx950): one block per
// (page, kv head), the transposed V page and then the slice-blocked K page.
//
// Replaces the FlashInfer window port's single-request decode
// (single_decode_with_kv_cache_with_jit_module(..., maybe_zhi_slice=...),
// kernels/flashinfer_port/fiwin_common.py:96-112, e2e_pipeline/atflash_e2e_fafi.py:106-109;
// window predicate: kernels/flashinfer_port/decode.cuh.diff:47-89).
//
// decode_kernel: one workgroup of 8 waves per (sequence, kv head, split of pages);
// each wave streams its own pages.  decode_wave_kernel: a workgroup per wave, for
// large batches.  decode_rows_kernel: the same decode over contiguous K and V rows
// in place of pages.  All three give the same bits.
//
// The G = Hq/Hkv query heads of the kv head are the 16 columns of
// v_mfma_f32_16x16x32_bf16 (S^T = K Q^T, four 8-dim slices per instruction) and
// v_mfma_f32_16x16x16_bf16 (O^T = V^T P^T, 16 tokens per instruction).  K and V are loaded straight into the MFMA operand registers.
// The window table is per 8-dim slice (16 entries; a 16-dim level table is
// passed as each level's value for its two slices).  Page p is read for the
// first n(p) = #{s : zhi8[s] >= (N-1) - (16p+15)} slices, those its youngest
// key reads: the page's K buffer range covers those slices only, so the loads
// of the other slices return zeros without a memory request and out-of-window
// K bytes are not read from HBM.  Page rule (level table, block_n = 16): every
// key of the page uses those slices.  Per-key rule (vec8 table, as the
// FlashInfer port's decode, kernels/flashinfer_port/decode.cuh.diff:47-89):
// on a page with a slice boundary inside it, an older key's out-of-window
// slices are zeroed in registers before the MFMA.
//
// Merging: the 8 wave partials (m, l, o) of a split are combined in LDS.  With
// one split per (sequence, kv head) the workgroup writes the output itself.
// Otherwise it stores the split's partial in the workspace and ends, and a
// second kernel (decode_merge_kernel, eight workgroups per (sequence, kv head))
// merges the split partials by log-sum-exp and writes the output.
// (decode_wave_kernel stores wave partials, which its merge kernels combine into
// the split's first.)  The kernel boundary orders the partial stores before the
// merge loads, so no workgroup waits on another inside a launch: no arrival
// counters, atomics or fences.
// (Measured against merging in the last-arriving workgroup of one launch: the
// chain store -> wait -> arrival atomic -> acquire -> loads there kept a single
// workgroup busy for about 7 us after the last split finished.)
#include <mutex>

#include "atf_decode_common.h"

namespace atf {

struct PageRegs {
  u32x4 k[4];  // slice quads (32 dims each)
  u32x2 v[8];  // 16-row d blocks
  int n0;
  bool mask;   // per-key rule with a slice boundary inside the page
};

// K and V operands of page p whose page-table entry is `raw`, reading its first
// ns slices of K; a page outside the split (in_split false) reads nothing.
// The page's V and K halves are range-checked buffer resources: a load at or
// past the range returns zeros without a memory request.  K's slices are a
// contiguous prefix of its half, so a range of ns * 256 bytes reads the
// in-window slices and yields zeros for the others, and what the page reads is
// one contiguous run (V, then those slices); an invalid page entry gets an
// empty range.  The loads are therefore unconditional: wave-uniform base,
// 32-bit lane offset, immediate row offset, no per-load address arithmetic.
// Every page is read once per call, so the loads are non-temporal.
// (The range goes through readfirstlane: the level count is uniform, but the
// compiler may count it in a vector register, and a resource built from one
// becomes a loop over lanes around every load.)
struct PageRef {
  size_t blk_elems;  // offset of the (page, kv head) block in the cache, in elements
  bool ok;
};
__device__ __forceinline__ PageRef page_ref(const DecHot& a, int h, int raw, bool in_split) {
  const int pg = __builtin_amdgcn_readfirstlane(raw);
  const bool ok = in_split && pg >= 0 && pg < a.num_pages;
  return PageRef{(static_cast<size_t>(ok ? pg : 0) * a.hkv + h) * kKvBlockElems, ok};
}
// K: slice 4 lp + lane/16, token lane%16: quad lp is the 1 KB run at lp * 1024
__device__ __forceinline__ void dec_load_k(const DecHot& a, const PageRef& pr, int ns, int lane, u32x4 (&k)[4]) {
  const int k_range = __builtin_amdgcn_readfirstlane(pr.ok ? ns * (kPage * kSliceDims * 2) : 0);
  const __amdgpu_buffer_rsrc_t rk =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.kv_cache) + pr.blk_elems + kKHalfElems, 0, k_range,
                                        kBufferWord3);
  const uint32_t koff = static_cast<uint32_t>(lane) << 4;
#pragma unroll
  for (int lp = 0; lp < 4; ++lp)
    k[lp] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, koff + lp * 1024u, 0, kLoadStream));
}
// V^T operand: d row 16*db + lane%16, tokens 4*(lane/16)..+3 -> stored slots.
__device__ __forceinline__ void dec_load_v(const DecHot& a, const PageRef& pr, int lane, u32x2 (&v)[8]) {
  const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(a.kv_cache) + pr.blk_elems, 0, pr.ok ? kBlockElems * 2 : 0, kBufferWord3);
  const int grp = lane >> 4;
  const int slot0 = 4 * ((grp == 1) ? 2 : (grp == 2 ? 1 : grp));
  const uint32_t voff = (static_cast<uint32_t>(lane & 15) << 5) + static_cast<uint32_t>(slot0) * 2u;
#pragma unroll
  for (int db = 0; db < 8; ++db)
    v[db] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rv, voff + db * 512u, 0, kLoadStream));
}
__device__ __forceinline__ void dec_load_page(const DecHot& a, int h, int raw, bool in_split, int p, int ns,
                                              bool mask, int lane, PageRegs& r) {
  r.n0 = p * kPage;
  r.mask = mask;
  const PageRef ref = page_ref(a, h, raw, in_split);
  dec_load_k(a, ref, ns, lane, r.k);
  dec_load_v(a, ref, lane, r.v);
}

// Decode of one split (pages `ord`) of sequence b: this wave's pages (kWaves waves
// take the split), its partial (m, l, o) to row `wave` of sh_o, sh_m and sh_l.
// ent: the page-table entries of the wave's first group.
template <bool kPerKey, int kWaves>
__device__ __forceinline__ void decode_pages(const DecHot& hot, const DecodeArgs& a, int h, int b, int N,
                                             const int32_t* row, const PageOrder& ord, int wave, int p_first,
                                             int (&ent)[kDecUnroll], float* sh_o, float* sh_m, float* sh_l) {
  constexpr int kStride = kDecUnroll * kWaves;
  const int p_end = ord.count, po = ord.po, pm = ord.pm;
  const int lane = threadIdx.x & 63, g = lane & 15;
  const float NEG_INF = -__builtin_huge_valf();
  const float c = a.scale_log2;

  // The first group's page loads are issued before Q is loaded and rotated, so
  // the wave's first memory round trip overlaps the Q work.  Each page's
  // registers are reloaded with the page one stride on right after the page is
  // used, so the next group's loads go out while the rest of the group is
  // computed.  (A group still starts with a wait for all of its loads: the
  // reloads are conditional on the split's end.  Issuing every load on every
  // path, so that each page is waited for with the later pages' loads still in
  // flight, measured slower.)
  PageRegs pr[kDecUnroll];
  // per-key rule: lane s < 16 holds zhi8[s], the others a limit no age meets,
  // so a page's slice counts are one compare and a ballot popcount each
  int zc = INT32_MIN;
#pragma unroll
  for (int s = 0; s < kSlices && kPerKey; ++s)
    if (lane == s) zc = a.st.zhi[s];
  // Straight-line code up to the first page loads (a page past the split gets
  // an empty buffer range: its loads return zeros without a memory request), so
  // the compiler reads every kernel argument they need in the first batch.
#pragma unroll
  for (int u = 0; u < kDecUnroll; ++u) {
    int ns;
    bool mask;
    page_slices<kPerKey>(a, zc, po + pm * (p_first + u), N, ns, mask);
    dec_load_page(hot, h, ent[u], p_first + u < p_end, po + pm * (p_first + u), ns, mask, lane, pr[u]);
  }
#pragma unroll
  for (int u = 0; u < kDecUnroll; ++u) ent[u] = dec_fetch_entry(row, ord, p_first + kStride + u);

  // ---- Q^T fragments: lane holds q head g, slice 4 lp + lane/16 ----
  // Every Q and (cos, sin) load is issued before any is used (one memory round
  // trip, not one per slice): lanes past the group read the group's last head
  // and a sequence of length 0 reads position 0, both in bounds, and are
  // zeroed afterwards.
  u32x4 Qf[4];
  {
    const int qh = h * a.group + min(g, a.group - 1);
    const bool valid = g < a.group && N > 0;
    const uint16_t* qrow = a.q + static_cast<int64_t>(b) * a.q_sb + static_cast<int64_t>(qh) * a.q_sh;
    load_slices4<4>(qrow, a.layout, lane >> 4, Qf);
    if (a.rope_cs != nullptr) {
      float cs[4][8];
#pragma unroll
      for (int lp = 0; lp < 4; ++lp) load_cs4(a.rope_cs, max(N - 1, 0), slice_pair0(4 * lp + (lane >> 4)), cs[lp]);
#pragma unroll
      for (int lp = 0; lp < 4; ++lp) Qf[lp] = rope_slice(Qf[lp], cs[lp]);
    }
#pragma unroll
    for (int lp = 0; lp < 4; ++lp)
      if (!valid) Qf[lp] = u32x4{0u, 0u, 0u, 0u};
  }
  // per-key rule: the distance limit of this lane's slice in each quad
  int zl[4] = {0, 0, 0, 0};
#pragma unroll
  for (int lp = 0; lp < 4 && kPerKey; ++lp) {
    const int sg = lane >> 4;
    const int z0 = a.st.zhi[4 * lp], z1 = a.st.zhi[4 * lp + 1], z2 = a.st.zhi[4 * lp + 2], z3 = a.st.zhi[4 * lp + 3];
    zl[lp] = sg == 0 ? z0 : (sg == 1 ? z1 : (sg == 2 ? z2 : z3));
  }

  f32x4 O[8];
#pragma unroll
  for (int db = 0; db < 8; ++db) O[db] = f32x4{};
  float m_run = NEG_INF, l_run = 0.f;

  for (int p0 = p_first; p0 < p_end; p0 += kStride) {
#pragma unroll
    for (int u = 0; u < kDecUnroll; ++u) {
      if (p0 + u >= p_end) break;
      PageRegs& r = pr[u];
      if (kPerKey && r.mask) {
        // a slice boundary inside the page: a key older than its slice's limit
        // (age > zhi8[slice]) drops that slice (lane: key lane%16, slice 4 lp + lane/16)
        const int age = (N - 1) - (r.n0 + (lane & 15));
#pragma unroll
        for (int lp = 0; lp < 4; ++lp)
          if (age > zl[lp]) r.k[lp] = u32x4{0u, 0u, 0u, 0u};
      }
      // all four slice quads: the out-of-window slices were loaded as zeros and
      // add exact zeros (cheaper than branching around their MFMAs)
      f32x4 S = f32x4{};
#pragma unroll
      for (int lp = 0; lp < 4; ++lp)
        S = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, r.k[lp]),
                                                    __builtin_bit_cast(bf16x8, Qf[lp]), S, 0, 0, 0);
      // S lane layout: q head g, tokens 4*(lane/16) + i.
      const int tok0 = r.n0 + 4 * (lane >> 4);
      const bool tail = r.n0 + kPage > N;
      // This page's registers take the page one stride on: K as soon as the QK
      // MFMAs have read it, V after the PV MFMAs (-0.46 us per call at 128K
      // against reloading both after the page, same box; outputs bitwise equal).
      const int pn = p0 + kStride + u;
      const bool reload = pn < p_end;
      bool mask_n = false;
      PageRef ref_n{0, false};
      if (reload) {
        int ns;
        page_slices<kPerKey>(a, zc, po + pm * pn, N, ns, mask_n);
        ref_n = page_ref(hot, h, ent[u], true);
        dec_load_k(hot, ref_n, ns, lane, r.k);
      }
      float mx = NEG_INF;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (tail && tok0 + i >= N) S[i] = NEG_INF;
        mx = fmaxf(mx, S[i]);
      }
      if (tail) {
        // zero V of tokens past N so that 0 * V stays 0
#pragma unroll
        for (int db = 0; db < 8; ++db) {
          if (tok0 + 0 >= N) r.v[db][0] &= 0xffff0000u;
          if (tok0 + 1 >= N) r.v[db][0] &= 0x0000ffffu;
          if (tok0 + 2 >= N) r.v[db][1] &= 0xffff0000u;
          if (tok0 + 3 >= N) r.v[db][1] &= 0x0000ffffu;
        }
      }
      mx = quad_max(mx);
      // Lazy reference max: m_run moves only where a score exceeds it by more
      // than 8 (log2 units; the first finite score always does), so P <= 256
      // and O and l are rescaled on few pages.
      const bool grow = (mx - m_run) * c > 8.f;  // -inf - -inf = NaN: no
      if (__builtin_amdgcn_ballot_w64(grow) != 0) {
        const float alpha = !grow ? 1.f : (m_run == NEG_INF ? 0.f : fast_exp2((m_run - mx) * c));
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < 8; ++db) O[db] *= alpha;
        m_run = grow ? mx : m_run;
      }
      const float msc = (m_run == NEG_INF) ? 0.f : m_run * c;
      float pv[4];
      float ls = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pv[i] = fast_exp2(__builtin_fmaf(S[i], c, -msc));
        ls += pv[i];
      }
      l_run += ls;
      u32x2 pk;
      pk[0] = pack_bf16x2(pv[0], pv[1]);
      pk[1] = pack_bf16x2(pv[2], pv[3]);
      const s16x4 pb = __builtin_bit_cast(s16x4, pk);
#pragma unroll
      for (int db = 0; db < 8; ++db)
        O[db] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, r.v[db]), pb, O[db], 0, 0, 0);
      if (reload) {
        dec_load_v(hot, ref_n, lane, r.v);
        r.n0 = (po + pm * pn) * kPage;
        r.mask = mask_n;
        ent[u] = dec_fetch_entry(row, ord, pn + kStride);
      }
    }
  }

  // ---- the split's partial: combine the wave partials in LDS ----
  const float l_tot = quad_sum(l_run);
  if (g < a.group) {
#pragma unroll
    for (int db = 0; db < 8; ++db) {
      const int d = 16 * db + 4 * (lane >> 4);
      *reinterpret_cast<f32x4*>(&sh_o[(wave * kDecMaxGroup + g) * kD + d]) = O[db];
    }
    if (lane < 16) {
      sh_m[wave * kDecMaxGroup + g] = m_run;
      sh_l[wave * kDecMaxGroup + g] = l_tot;
    }
  }
}

// two waves per SIMD: at most 256 registers per wave.  kWaves = 8 (one
// workgroup per CU) or 4 (short contexts: smaller splits over more CUs).
template <bool kPerKey, int kWaves>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2)))
void decode_kernel(const int32_t* page_table, const int32_t* seq_lens, const uint16_t* kv_cache, int max_pages,
                   int pages_per_split, int max_seq_len, int hkv, int num_pages, int n_splits, DecodeArgs a) {
  const DecHot hot{page_table, seq_lens, kv_cache, max_pages, pages_per_split, max_seq_len, hkv, num_pages, n_splits};
  // wave partials
  __shared__ __attribute__((aligned(16))) float sh_o[kWaves * kDecMaxGroup * kD];
  __shared__ float sh_m[kWaves * kDecMaxGroup], sh_l[kWaves * kDecMaxGroup];

  const int s = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x;
  const int wave = tid >> 6;
  // Local page indices: wave w takes the groups of kDecUnroll local pages that
  // start at kDecUnroll * (w + kWaves * i); local page j is page po + pm * j.
  const int p_first = kDecUnroll * __builtin_amdgcn_readfirstlane(wave);
  PageOrder ord = page_order(s, hot.n_splits, hot.pages_per_split);
  const int po = ord.po, pm = ord.pm;
  // The first group's page-table entries are fetched together with the
  // sequence length, their index clamped into the table row only (an entry
  // past the split is never used), so the first page loads wait for two
  // memory round trips after the kernel arguments, not three.
  int ent[kDecUnroll];
  const int32_t* row = hot.page_table + static_cast<int64_t>(b) * hot.max_pages;
#pragma unroll
  for (int u = 0; u < kDecUnroll; ++u) ent[u] = row[min(po + pm * (p_first + u), hot.max_pages - 1)];
  const int N = max(0, min(hot.seq_lens[b], hot.max_seq_len));
  const int n_pages = (N + kPage - 1) / kPage;
  set_page_count(ord, s, hot.n_splits, hot.pages_per_split, n_pages);
  decode_pages<kPerKey, kWaves>(hot, a, h, b, N, row, ord, wave, p_first, ent, sh_o, sh_m, sh_l);
  __syncthreads();
  store_split<kWaves>(a, (static_cast<int64_t>(b) * hot.hkv + h) * a.n_splits + s, a.n_splits == 1, h, b, sh_o, sh_m, sh_l);
}

// ---- a batch spread over the chip wave by wave ----
// decode_kernel's grid gives every sequence of a batch the splits of the longest
// one, as many as fit 256 workgroups, and a workgroup keeps a split's eight waves
// on one CU: a ragged batch leaves most CUs with little to do while a few stream
// the long sequences, and sequence x kv head counts that do not divide 256 start a
// second wave of workgroups.  Here every wave of every split is a workgroup of its
// own, so that the waves of a long sequence spread over all CUs; where there are
// more of them than the chip holds (eight a CU), those of the longest sequences
// are dispatched first.  The lengths live in device memory: a wave finds the
// sequence that its place in the grid means from them.
// Pages, page order and arithmetic of a wave are decode_kernel's, and
// decode_wave_merge_kernel combines waves and splits in decode_kernel's and
// decode_merge_kernel's order: the outputs are theirs bit for bit, whatever the
// other sequences of the batch hold.
//   HBM bound.  Against decode_kernel and its merge on the same batch (24 / 8
// heads, vec8 k = 2; us a call): 12 sequences of 700 to 32768 tokens 110.8 -> 69.8,
// 40 of 300 to 9000 (level table) 99.3 -> 67.3, 12 of 32768 261 -> 207, 40 of 8192
// 210 -> 177, 8 of 32768 124.5 -> 123.4.  At 168 registers, three waves a SIMD, the
// page registers spill: 12 ragged sequences 274.
// grid: x = split, y = kv head + kv heads x wave, z = the sequence, or its rank by
// length (a.by_length).  Pages that lie side by side, and a page's blocks of the kv
// heads, are then read at about the same time: with the waves of a split before
// the heads 32 x 16K tokens take 280 us and not 261 (24 / 8 heads, vec8 k = 2), with
// heads and waves before the splits 4 x 128K 196 and not 176 (28 / 4 heads, OFF).
template <bool kPerKey>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2)))
void decode_wave_kernel(const int32_t* page_table, const int32_t* seq_lens, const uint16_t* kv_cache, int max_pages,
                        int pages_per_split, int max_seq_len, int hkv, int num_pages, int n_splits, DecodeArgs a) {
  const DecHot hot{page_table, seq_lens, kv_cache, max_pages, pages_per_split, max_seq_len, hkv, num_pages, n_splits};
  const int s = blockIdx.x, h = blockIdx.y % hkv, wave = blockIdx.y / hkv;
  int b = blockIdx.z;
  if (a.by_length) b = a.batch <= 64 ? nth_longest<1>(seq_lens, a.batch, max_seq_len, b)
                                     : nth_longest<kDecSpreadBatch / 64>(seq_lens, a.batch, max_seq_len, b);
  const int p_first = kDecUnroll * wave;
  PageOrder ord = page_order(s, n_splits, pages_per_split);
  int ent[kDecUnroll];
  const int32_t* row = page_table + static_cast<int64_t>(b) * max_pages;
#pragma unroll
  for (int u = 0; u < kDecUnroll; ++u) ent[u] = row[min(ord.po + ord.pm * (p_first + u), max_pages - 1)];
  const int N = max(0, min(seq_lens[b], max_seq_len));
  set_page_count(ord, s, n_splits, pages_per_split, (N + kPage - 1) / kPage);
  // wave partials: o [(sequence, kv head, split, wave)][group][128], then m [group] and l [group] of each
  const int64_t unit = ((static_cast<int64_t>(b) * hkv + h) * n_splits + s) * kDecWaves + wave;
  float* ml = a.ws_ml + unit * 2 * a.group;
  decode_pages<kPerKey, kDecWaves>(hot, a, h, b, N, row, ord, 0, p_first, ent, a.ws_o + unit * a.group * kD, ml,
                                   ml + a.group);
}

// ---- decode over contiguous K and V rows ----
// The same decode reading a sequence's K and V as rows [token][128] with strides,
// as the reference's decode call passes them, instead of a paged cache: K
// (rotated here when rope_cs is given) and V are read once, where packing them
// into pages first reads them, writes them and reads them again.  Blocks of 16
// tokens take the place of pages, and everything else (window rules, splits,
// waves, MFMA operands, merge) is decode_kernel's, so the outputs are those of
// the packed cache bit for bit.
//   K: lane (token t = lane % 16, g = lane / 16) reads slices g, 4 + g, 8 + g and
// 12 + g of its token's row: 16 bytes each (sorted-pair rows), or 8 + 8 (the two
// halves of the slice's pairs in half-split rows).  A slice past the page's
// window, or of a token past the sequence, is read at an offset past the buffer
// range: zeros, no request.
//   V: lane (g, i = lane % 16) reads dims 8i..8i+7 of tokens 4g..4g+3 (16 lanes
// read whole 256-byte rows); MFMA e takes element e of each, four tokens deep,
// so its row i is dim 8i + e and the transposition is two byte permutes per MFMA.
//   HBM bound.  Against the call that packs first (28 / 4 heads, k = 2, pre-rotated
// rows): 32K tokens 71.2 -> 18.6 us (26.5 us of writer, 18.5 us of decode and
// merge, and the host's allocations and copies before); 128K OFF 50.9 us a call.
struct RowsArgs {
  DecodeArgs d;  // page fields unused; d.max_seq_len is the length of every sequence
  DecodeRows r;
};

constexpr uint32_t kRowsRange = 0x7fffffffu;  // buffer range of a block's rows
constexpr uint32_t kRowsSkip = 0x80000000u;   // an offset past it

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, static_cast<int>(kRowsRange), kBufferWord3);
}

template <bool kRope>
struct RowBlock {
  u32x4 k[4];
  u32x4 v[4];
  u32x4 cs[kRope ? 8 : 1];  // (cos, sin) of the four slices' pairs
};

// kHalf: half-split rows (kRope implies it), otherwise sorted-pair rows.
// kU: blocks in flight per wave (with RoPE two: their (cos, sin) take as many
// registers as K and V).
template <bool kPerKey, bool kHalf, bool kRope, int kWaves>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2)))
void decode_rows_kernel(RowsArgs ra) {
  constexpr int kU = kRope ? 2 : 4;
  static_assert(kDecUnroll % kU == 0 && (kHalf || !kRope), "rows kernel");
  const DecodeArgs& a = ra.d;
  __shared__ __attribute__((aligned(16))) float sh_o[kWaves * kDecMaxGroup * kD];
  __shared__ float sh_m[kWaves * kDecMaxGroup], sh_l[kWaves * kDecMaxGroup];
  const int s = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int g = lane >> 4, t = lane & 15;
  const int N = a.max_seq_len;
  PageOrder ord = page_order(s, a.n_splits, a.pages_per_split);
  set_page_count(ord, s, a.n_splits, a.pages_per_split, (N + kPage - 1) / kPage);
  const float NEG_INF = -__builtin_huge_valf();
  const float c = a.scale_log2;
  // the wave's blocks in decode_kernel's order: block j of the wave is local
  // page kDecUnroll (w + kWaves (j / kDecUnroll)) + j % kDecUnroll of the split
  auto local = [&](int j) { return kDecUnroll * (wave + kWaves * (j / kDecUnroll)) + j % kDecUnroll; };

  const uint8_t* kbase = reinterpret_cast<const uint8_t*>(ra.r.k + b * ra.r.ks_b + h * ra.r.ks_h);
  const uint8_t* vbase = reinterpret_cast<const uint8_t*>(ra.r.v + b * ra.r.vs_b + h * ra.r.vs_h);
  const int64_t kt = 2 * ra.r.ks_t, vt = 2 * ra.r.vs_t;  // bytes per token
  uint32_t koff[4];
  int zl[4];  // distance limits of the lane's slices (page rule: level 0 has none)
#pragma unroll
  for (int lp = 0; lp < 4; ++lp) {
    const int sl = 4 * lp + g;
    koff[lp] = static_cast<uint32_t>(t * kt) + 2 * (kHalf ? slice_pair0(sl) : 8 * sl);
    zl[lp] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (g == i) zl[lp] = (!kPerKey && 4 * lp + i < 2) ? INT32_MAX : a.st.zhi[4 * lp + i];
  }

  auto load_k = [&](int p, RowBlock<kRope>& r) {
    const int n0 = p * kPage;
    const int z = max(0, (N - 1) - (n0 + kPage - 1));  // the youngest key's age
    const auto rk = rows_rsrc(kbase + n0 * kt);
    const bool in = n0 + t < N;
#pragma unroll
    for (int lp = 0; lp < 4; ++lp) {
      const bool on = in && zl[lp] >= z;
      if constexpr (kHalf) {
        const u32x2 x1 = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_raw_buffer_load_b64(rk, on ? koff[lp] : kRowsSkip, 0, kLoadStream));
        const u32x2 x2 = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_raw_buffer_load_b64(rk, on ? koff[lp] + 2 * kP : kRowsSkip, 0, kLoadStream));
        r.k[lp] = u32x4{x1[0], x1[1], x2[0], x2[1]};
      } else {
        r.k[lp] = __builtin_bit_cast(
            u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, on ? koff[lp] : kRowsSkip, 0, kLoadStream));
      }
    }
    if constexpr (kRope) {
      const auto rc = rows_rsrc(a.rope_cs + static_cast<int64_t>(n0) * (2 * kP));
#pragma unroll
      for (int lp = 0; lp < 4; ++lp) {
        const bool on = in && zl[lp] >= z;
        const uint32_t off = t * (kP * 8) + slice_pair0(4 * lp + g) * 8;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          r.cs[2 * lp + i] = __builtin_bit_cast(
              u32x4, __builtin_amdgcn_raw_buffer_load_b128(rc, on ? off + 16 * i : kRowsSkip, 0, 0));
      }
    }
  };
  auto load_v = [&](int p, RowBlock<kRope>& r) {
    const int n0 = p * kPage;
    const auto rv = rows_rsrc(vbase + n0 * vt);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t off = static_cast<uint32_t>((4 * g + i) * vt) + 16 * t;
      r.v[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                             rv, n0 + 4 * g + i < N ? off : kRowsSkip, 0, kLoadStream));
    }
  };
  RowBlock<kRope> blk[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u)
    if (local(u) < ord.count) {
      const int p = ord.po + ord.pm * local(u);
      load_k(p, blk[u]);
      load_v(p, blk[u]);
    }

  // Q as decode_kernel loads it
  u32x4 Qf[4];
  {
    const int qh = h * a.group + min(t, a.group - 1);
    const uint16_t* qrow = a.q + b * a.q_sb + qh * a.q_sh;
    load_slices4<4>(qrow, kHalf ? kLayoutHalfSplit : kLayoutSortedPair, g, Qf);
    if constexpr (kRope) {
#pragma unroll
      for (int lp = 0; lp < 4; ++lp) {
        float cs[8];
        load_cs4(a.rope_cs, N - 1, slice_pair0(4 * lp + g), cs);
        Qf[lp] = rope_slice(Qf[lp], cs);
      }
    }
#pragma unroll
    for (int lp = 0; lp < 4; ++lp)
      if (t >= a.group) Qf[lp] = u32x4{0u, 0u, 0u, 0u};
  }

  f32x4 O[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) O[e] = f32x4{};
  float m_run = NEG_INF, l_run = 0.f;
  for (int j0 = 0; local(j0) < ord.count; j0 += kU) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (local(j0 + u) >= ord.count) break;
      RowBlock<kRope>& r = blk[u];
      const int n0 = (ord.po + ord.pm * local(j0 + u)) * kPage;
      // slices past the window: of the key (per-key rule) or of the page's youngest key
      const int age = kPerKey ? (N - 1) - (n0 + t) : max(0, (N - 1) - (n0 + kPage - 1));
      f32x4 S = f32x4{};
#pragma unroll
      for (int lp = 0; lp < 4; ++lp) {
        u32x4 K = r.k[lp];
        if constexpr (kRope) {
          float cs[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) cs[i] = __uint_as_float(r.cs[2 * lp + (i >> 2)][i & 3]);
          K = rope_slice(K, cs);
        }
        if (age > zl[lp]) K = u32x4{0u, 0u, 0u, 0u};
        S = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, K), __builtin_bit_cast(bf16x8, Qf[lp]), S, 0,
                                                    0, 0);
      }
      const int jn = local(j0 + kU + u);
      const bool reload = jn < ord.count;
      if (reload) load_k(ord.po + ord.pm * jn, r);
      // S: query head lane % 16, tokens 4 (lane / 16) + i
      float mx = NEG_INF;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (n0 + 4 * g + i >= N) S[i] = NEG_INF;
        mx = fmaxf(mx, S[i]);
      }
      mx = quad_max(mx);
      const bool grow = (mx - m_run) * c > 8.f;  // the lazy reference max of decode_kernel
      if (__builtin_amdgcn_ballot_w64(grow) != 0) {
        const float alpha = !grow ? 1.f : (m_run == NEG_INF ? 0.f : fast_exp2((m_run - mx) * c));
        l_run *= alpha;
#pragma unroll
        for (int e = 0; e < 8; ++e) O[e] *= alpha;
        m_run = grow ? mx : m_run;
      }
      const float msc = (m_run == NEG_INF) ? 0.f : m_run * c;
      float pv[4];
      float ls = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pv[i] = fast_exp2(__builtin_fmaf(S[i], c, -msc));
        ls += pv[i];
      }
      l_run += ls;
      const s16x4 pb = __builtin_bit_cast(s16x4, u32x2{pack_bf16x2(pv[0], pv[1]), pack_bf16x2(pv[2], pv[3])});
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t sel = (e & 1) ? 0x07060302u : 0x05040100u;  // the odd or even halves of two words
        const u32x2 col = {__builtin_amdgcn_perm(r.v[1][e >> 1], r.v[0][e >> 1], sel),
                           __builtin_amdgcn_perm(r.v[3][e >> 1], r.v[2][e >> 1], sel)};
        O[e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, col), pb, O[e], 0, 0, 0);
      }
      if (reload) load_v(ord.po + ord.pm * jn, r);
    }
  }

  const float l_tot = quad_sum(l_run);
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
  store_split<kWaves>(a, (static_cast<int64_t>(b) * a.hkv + h) * a.n_splits + s, a.n_splits == 1, h, b, sh_o, sh_m, sh_l);
}

// ---- measurement probe: the streaming ceiling of the decode's page loads ----
// decode_kernel's grid, waves, split rule, page-table fetches and page loads
// (the same range-checked, non-temporal buffer loads of V and of the K slices
// the page's youngest key reads under a.st, the same 4-page groups with the
// rolling reload), with the compute replaced by an XOR of the loaded words, no
// LDS combine and no merge: what the memory system delivers to this access
// pattern.  One word per wave goes to
// sink[((b * hkv + h) * n_splits + s) * kDecWaves + wave].
__global__ __launch_bounds__(kDecWaves * 64) __attribute__((amdgpu_waves_per_eu(2)))
void decode_stream_probe_kernel(const int32_t* page_table, const int32_t* seq_lens, const uint16_t* kv_cache,
                                int max_pages, int pages_per_split, int max_seq_len, int hkv, int num_pages,
                                int n_splits, uint32_t* sink, DecodeArgs a) {
  const DecHot hot{page_table, seq_lens, kv_cache, max_pages, pages_per_split, max_seq_len, hkv, num_pages, n_splits};
  const int s = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x;
  const int wave = tid >> 6, lane = tid & 63;
  constexpr int kStride = kDecUnroll * kDecWaves;
  const int p_first = kDecUnroll * __builtin_amdgcn_readfirstlane(wave);
  PageOrder ord = page_order(s, hot.n_splits, hot.pages_per_split);
  const int po = ord.po, pm = ord.pm;
  int ent[kDecUnroll];
  const int32_t* row = hot.page_table + static_cast<int64_t>(b) * hot.max_pages;
#pragma unroll
  for (int u = 0; u < kDecUnroll; ++u) ent[u] = row[min(po + pm * (p_first + u), hot.max_pages - 1)];
  const int N = max(0, min(hot.seq_lens[b], hot.max_seq_len));
  const int n_pages = (N + kPage - 1) / kPage;
  set_page_count(ord, s, hot.n_splits, hot.pages_per_split, n_pages);
  const int p_end = ord.count;
  PageRegs pr[kDecUnroll];
  int zc = INT32_MIN;
#pragma unroll
  for (int sl = 0; sl < kSlices; ++sl)
    if (lane == sl) zc = a.st.zhi[sl];
#pragma unroll
  for (int u = 0; u < kDecUnroll; ++u) {
    int ns;
    bool mask;
    page_slices<true>(a, zc, po + pm * (p_first + u), N, ns, mask);
    dec_load_page(hot, h, ent[u], p_first + u < p_end, po + pm * (p_first + u), ns, false, lane, pr[u]);
  }
#pragma unroll
  for (int u = 0; u < kDecUnroll; ++u) ent[u] = dec_fetch_entry(row, ord, p_first + kStride + u);
  uint32_t acc = 0;
  for (int p0 = p_first; p0 < p_end; p0 += kStride) {
#pragma unroll
    for (int u = 0; u < kDecUnroll; ++u) {
      if (p0 + u >= p_end) break;
      PageRegs& r = pr[u];
#pragma unroll
      for (int lp = 0; lp < 4; ++lp) acc ^= r.k[lp][0] ^ r.k[lp][1] ^ r.k[lp][2] ^ r.k[lp][3];
#pragma unroll
      for (int db = 0; db < 8; ++db) acc ^= r.v[db][0] ^ r.v[db][1];
      const int pn = p0 + kStride + u;
      if (pn < p_end) {
        int ns;
        bool mask;
        page_slices<true>(a, zc, po + pm * pn, N, ns, mask);
        dec_load_page(hot, h, ent[u], true, po + pm * pn, ns, false, lane, pr[u]);
        ent[u] = dec_fetch_entry(row, ord, pn + kStride);
      }
    }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) acc ^= static_cast<uint32_t>(__shfl_xor(static_cast<int>(acc), m));
  if (lane == 0) sink[((static_cast<int64_t>(b) * hkv + h) * n_splits + s) * kDecWaves + wave] = acc;
}

// ---- merge ----
__global__ __launch_bounds__(512) void decode_merge_kernel(const float* ws_ml, const float* ws_o, uint16_t* out,
                                                           int64_t o_sb, int64_t o_sh, int n_splits, int group,
                                                           int hkv, float scale_log2) {
  merge_splits<false>(MergeArgs{ws_ml, ws_o, out, o_sb, o_sh, n_splits, group, hkv, scale_log2}, n_splits);
}

// The merge after decode_wave_kernel: eight wave partials a split, then the splits.
__global__ __launch_bounds__(512) void decode_wave_merge_kernel(const float* ws_ml, const float* ws_o, uint16_t* out,
                                                                int64_t o_sb, int64_t o_sh, int n_splits, int group,
                                                                int hkv, float scale_log2) {
  merge_splits<true>(MergeArgs{ws_ml, ws_o, out, o_sb, o_sh, n_splits, group, hkv, scale_log2}, n_splits);
}

// The same for at most kSplits (1 or 4) splits, without idle lanes for the splits
// and heads that are not there: 4 kSplits lanes take 16 dims of a query head, the
// rows (sequence, query head, 16 dims) lie one after the other.  The sums are
// merge_splits', whose further exchanges meet empty partials here.
constexpr int kMergeFewThreads = 256;
template <int kSplits>
__global__ __launch_bounds__(kMergeFewThreads) void decode_wave_merge_few_kernel(
    const float* ws_ml, const float* ws_o, uint16_t* out, int64_t o_sb, int64_t o_sh, int n_splits, int group, int hkv,
    float scale_log2, int rows) {
  static_assert(kSplits == 1 || kSplits == 4, "one lane group, or the four of a 16-lane row");
  const MergeArgs a{ws_ml, ws_o, out, o_sb, o_sh, n_splits, group, hkv, scale_log2};
  const int t = blockIdx.x * kMergeFewThreads + threadIdx.x;
  const int row = t / (kMergeLanes * kSplits), sp = t / kMergeLanes % kSplits;
  const int md4 = row % kMergeChunks * kMergeDims + 4 * (t % kMergeLanes);
  const int head = row / kMergeChunks;                 // sequence, query head
  const int pair = head / group, mg = head % group;    // sequence, kv head
  float M = -__builtin_huge_valf(), L = 0.f;
  f32x4 acc = f32x4{};
  if (row < rows && sp < n_splits) load_wave_split(a, static_cast<int64_t>(pair) * n_splits + sp, mg, md4, M, L, acc);
  if constexpr (kSplits > 1) merge_rows(M, L, acc, scale_log2);
  if (row < rows && sp == 0) store_merged(a, pair / hkv, pair % hkv * group + mg, md4, L, acc);
}

// Level count per page for one sequence of length N under the page rule
// (block_n = 16), as page_slices<false> computes it (the kernel reads twice as
// many 8-dim slices).
__global__ void decode_page_levels_kernel(int32_t* out, int n_pages, int N, LevelTable lt) {
  const int p = blockIdx.x * blockDim.x + threadIdx.x;
  if (p >= n_pages) return;
  out[p] = levels_of(lt, max(0, (N - 1) - (p * kPage + kPage - 1)));
}

// The merge of a call's split partials (nothing to do with one split in one workgroup).
hipError_t launch_decode_merge(const DecodeArgs& a, hipStream_t s) {
  if (!a.spread && a.n_splits == 1) return hipSuccess;
  const float *ml = a.ws_ml, *o = a.ws_o;
  if (a.spread && a.n_splits <= 4) {
    const int rows = a.batch * a.hq * kMergeChunks, lanes = kMergeLanes * (a.n_splits == 1 ? 1 : 4);
    const dim3 grid((rows * lanes + kMergeFewThreads - 1) / kMergeFewThreads);
    hipLaunchKernelGGL(a.n_splits == 1 ? decode_wave_merge_few_kernel<1> : decode_wave_merge_few_kernel<4>, grid,
                       dim3(kMergeFewThreads), 0, s, ml, o, a.out, a.o_sb, a.o_sh, a.n_splits, a.group, a.hkv,
                       a.scale_log2, rows);
  } else {
    hipLaunchKernelGGL(a.spread ? decode_wave_merge_kernel : decode_merge_kernel, dim3(kMergeChunks, a.hkv, a.batch),
                       dim3(512), 0, s, ml, o, a.out, a.o_sb, a.o_sh, a.n_splits, a.group, a.hkv, a.scale_log2);
  }
  return hipGetLastError();
}

hipError_t launch_decode(const DecodeArgs& a, hipStream_t s) {
  if (a.batch <= 0) return hipSuccess;
  if (a.spread) {
#define ATF_WAVE_LAUNCH(PK)                                                                                        \
  hipLaunchKernelGGL(decode_wave_kernel<PK>, dim3(a.n_splits, a.hkv * kDecWaves, a.batch), dim3(64), 0, s,          \
                     a.page_table, a.seq_lens, a.kv_cache, a.max_pages, a.pages_per_split, a.max_seq_len, a.hkv,     \
                     a.num_pages, a.n_splits, a)
    if (a.per_key) ATF_WAVE_LAUNCH(true); else ATF_WAVE_LAUNCH(false);
#undef ATF_WAVE_LAUNCH
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    return launch_decode_merge(a, s);
  }
  const dim3 grid(a.n_splits, a.hkv, a.batch);
#define ATF_DEC_LAUNCH(PK, W)                                                                                   \
  hipLaunchKernelGGL((decode_kernel<PK, W>), grid, dim3(W * 64), 0, s, a.page_table, a.seq_lens, a.kv_cache,    \
                     a.max_pages, a.pages_per_split, a.max_seq_len, a.hkv, a.num_pages, a.n_splits, a)
  if (a.waves == 8) {
    if (a.per_key) ATF_DEC_LAUNCH(true, 8); else ATF_DEC_LAUNCH(false, 8);
  } else {
    if (a.per_key) ATF_DEC_LAUNCH(true, 4); else ATF_DEC_LAUNCH(false, 4);
  }
#undef ATF_DEC_LAUNCH
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  return launch_decode_merge(a, s);
}

hipError_t launch_decode_rows(const DecodeArgs& a, const DecodeRows& r, hipStream_t s) {
  if (a.batch <= 0) return hipSuccess;
  const dim3 grid(a.n_splits, a.hkv, a.batch);
  const RowsArgs ra{a, r};
#define ATF_ROWS_LAUNCH(PK, HALF, ROPE)                                                                  \
  do {                                                                                                   \
    if (a.waves == 8)                                                                                    \
      hipLaunchKernelGGL((decode_rows_kernel<PK, HALF, ROPE, 8>), grid, dim3(512), 0, s, ra);            \
    else                                                                                                 \
      hipLaunchKernelGGL((decode_rows_kernel<PK, HALF, ROPE, 4>), grid, dim3(256), 0, s, ra);            \
  } while (0)
  if (a.rope_cs != nullptr) {
    if (a.per_key) ATF_ROWS_LAUNCH(true, true, true); else ATF_ROWS_LAUNCH(false, true, true);
  } else if (a.layout == kLayoutHalfSplit) {
    if (a.per_key) ATF_ROWS_LAUNCH(true, true, false); else ATF_ROWS_LAUNCH(false, true, false);
  } else {
    if (a.per_key) ATF_ROWS_LAUNCH(true, false, false); else ATF_ROWS_LAUNCH(false, false, false);
  }
#undef ATF_ROWS_LAUNCH
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  return launch_decode_merge(a, s);
}

// ---- fixed scratch for the entry point that allocates nothing ----
// One copy per GPU, held until the process ends.  In host code `scratch` is a
// stand-in for the symbol, not a device address: kernels and copies take the
// address hipGetSymbolAddress returns for the current device, kept per device.
// It holds split partials only; nothing in it has to start at any value.
static __device__ __align__(256) uint8_t scratch[kDecScratchBytes];

namespace {
constexpr int kMaxDevices = 64;
std::mutex g_scratch_mu;
uint8_t* g_scratch_ptr[kMaxDevices];  // device address of `scratch` per device, null until looked up

// The current device's scratch, looked up on its first use on that device.
// That first use must not be under stream capture on `s` (the lookup is not a
// stream operation and may load the code object): it fails with
// hipErrorStreamCaptureUnsupported instead.
hipError_t device_scratch(uint8_t** out, hipStream_t s) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return hipErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (g_scratch_ptr[dev] == nullptr) {
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    e = hipStreamIsCapturing(s, &cs);
    if (e != hipSuccess) return e;
    if (cs != hipStreamCaptureStatusNone) return hipErrorStreamCaptureUnsupported;
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (e != hipSuccess) return e;
    if (p == nullptr) return hipErrorInvalidSymbol;
    g_scratch_ptr[dev] = static_cast<uint8_t*>(p);
  }
  *out = g_scratch_ptr[dev];
  return hipSuccess;
}
}  // namespace

hipError_t launch_decode_noalloc(DecodeArgs a, hipStream_t s) {
  if (a.batch <= 0) return hipSuccess;
  uint8_t* base = nullptr;
  hipError_t e = device_scratch(&base, s);
  if (e != hipSuccess) return e;
  a.ws_ml = reinterpret_cast<float*>(base);
  a.ws_o = a.ws_ml + static_cast<size_t>(a.batch) * a.hkv * a.n_splits * kDecMaxGroup * 2;
  return launch_decode(a, s);
}

hipError_t launch_decode_stream_probe(const DecodeArgs& a, uint32_t* sink, hipStream_t s) {
  if (a.batch <= 0) return hipSuccess;
  hipLaunchKernelGGL(decode_stream_probe_kernel, dim3(a.n_splits, a.hkv, a.batch), dim3(kDecWaves * 64), 0, s,
                     a.page_table, a.seq_lens, a.kv_cache, a.max_pages, a.pages_per_split, a.max_seq_len, a.hkv,
                     a.num_pages, a.n_splits, sink, a);
  return hipGetLastError();
}

hipError_t launch_decode_page_levels(int32_t* out, int n_pages, int seq_len, const LevelTable& lt,
                                     hipStream_t s) {
  if (n_pages <= 0) return hipSuccess;
  hipLaunchKernelGGL(decode_page_levels_kernel, dim3((n_pages + 255) / 256), dim3(256), 0, s, out, n_pages,
                     seq_len, lt);
  return hipGetLastError();
}

}  // namespace atf
