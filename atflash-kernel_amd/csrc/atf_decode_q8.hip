// Windowed split-KV decode over the paged cache of 8-bit floats: decode_kernel's
// attention with half its bytes.
//
// Mathematics.  A page's keys are K = code 2^eK and its values V = code 2^eV (e4m3
// codes, one exponent per page, kv head and half), so S = scale q K^T and O =
// softmax(S) V are formed as in decode_kernel once the codes have become bf16: e4m3
// has 4 significant bits and the scales are powers of two, so code 2^e is a bf16
// number exactly and nothing is rounded on the way (v_cvt_scalef32_pk_bf16_fp8: two
// codes times the scale an instruction).  Q keeps its bf16 precision, which a product
// on 8-bit operands would not leave it; the running maximum, the sum and O are fp32.
//
// Layout (atf_common.h): a page's block is 4 KB, V and then K, in the order in which
// the lanes of a wave take them: four loads of 16 bytes a lane, each 1 KB of
// consecutive bytes, bring in a whole page.
//   K: load j, lane (token t = lane % 16, g = lane / 16): the two slices of level
//      4j + g.  Slice i of it is the lane's share of MFMA 2j + i, whose 32 dims are
//      slice i of levels 4j .. 4j + 3.
//   V: load j, lane (row r, g): dims 8r + 4j .. + 3 of tokens 4g .. 4g + 3; dim d of them
//      is the lane's share of MFMA 4j + d, whose row r is dim 8r + 4j + d.
// The window shortens the K read to whole levels (256 bytes); a last odd slice is
// zeroed in registers with the per-key rule's.
#include "atf_decode_common.h"

namespace atf {

// Pages in flight per wave: their registers are half of a bf16 page's.  The order of
// a wave's pages is decode_kernel's, groups of kDecUnroll.
constexpr int kQ8Unroll = 8;
static_assert(kQ8Unroll % kDecUnroll == 0, "whole groups");

struct Q8Page {
  u32x4 k[2];
  u32x4 v[2];
  uint32_t e;  // eV | eK << 8
  int n0;
  bool mask;  // slices to zero by key
};

// Local page of the split that is the wave's i-th.
template <int kWaves>
__device__ __forceinline__ int q8_local(int wave, int i) {
  return kDecUnroll * (wave + kWaves * (i / kDecUnroll)) + i % kDecUnroll;
}

struct Q8Ref {
  size_t blk;  // index of the (page, kv head) block
  bool ok;
};
__device__ __forceinline__ Q8Ref q8_ref(const DecHot& hot, int h, int raw, bool in_split) {
  const int pg = __builtin_amdgcn_readfirstlane(raw);
  const bool ok = in_split && pg >= 0 && pg < hot.num_pages;
  return Q8Ref{static_cast<size_t>(ok ? pg : 0) * hot.hkv + h, ok};
}
// The first ns slices of K (whole levels) and the exponents; ranges as in decode_kernel:
// what lies past them is zero without a memory request.
__device__ __forceinline__ void q8_load_k(const DecHot& hot, const DecodeArgs& a, const Q8Ref& ref, int ns, int lane,
                                          Q8Page& p) {
  const uint8_t* base = reinterpret_cast<const uint8_t*>(hot.kv_cache) + ref.blk * kQ8BlockBytes + kQ8HalfBytes;
  const int range = __builtin_amdgcn_readfirstlane(ref.ok ? (ns + 1) / 2 * (kPage * 2 * kSliceDims) : 0);
  const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, range, kBufferWord3);
#pragma unroll
  for (int j = 0; j < 2; ++j)
    p.k[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, (static_cast<uint32_t>(lane) << 4) + j * 1024u,
                                                                             0, kLoadStream));
  const __amdgpu_buffer_rsrc_t re =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.kv_exps) + 2 * ref.blk, 0, ref.ok ? 2 : 0, kBufferWord3);
  p.e = static_cast<uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(re, 0, 0, 0));
}
__device__ __forceinline__ void q8_load_v(const DecHot& hot, const Q8Ref& ref, int lane, Q8Page& p) {
  const uint8_t* base = reinterpret_cast<const uint8_t*>(hot.kv_cache) + ref.blk * kQ8BlockBytes;
  const __amdgpu_buffer_rsrc_t rv =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, ref.ok ? kQ8HalfBytes : 0, kBufferWord3);
#pragma unroll
  for (int j = 0; j < 2; ++j)
    p.v[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, (static_cast<uint32_t>(lane) << 4) + j * 1024u,
                                                                             0, kLoadStream));
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

// The slices a page reads (page_slices), and whether some are to be zeroed by key: a
// boundary inside the page, or a last level of which only the first slice is read.
template <bool kPerKey>
__device__ __forceinline__ void q8_slices(const DecodeArgs& a, int zc, int p, int N, int& ns, bool& mask) {
  page_slices<kPerKey>(a, zc, p, N, ns, mask);
  if (kPerKey) mask = mask || (ns & 1) != 0;
}

// Decode of one split (pages `ord`) of sequence b: this wave's pages (kWaves waves
// take the split), its partial (m, l, o) to row `out` of sh_o, sh_m and sh_l.
template <bool kPerKey, int kWaves>
__device__ __forceinline__ void decode_pages_q8(const DecHot& hot, const DecodeArgs& a, int h, int b, int N,
                                                const int32_t* row, const PageOrder& ord, int wave, int out,
                                                int (&ent)[kQ8Unroll], float* sh_o, float* sh_m, float* sh_l) {
  const int count = ord.count, po = ord.po, pm = ord.pm;
  const int lane = threadIdx.x & 63, t = lane & 15, g = lane >> 4;
  const float NEG_INF = -__builtin_huge_valf();
  const float c = a.scale_log2;

  Q8Page pr[kQ8Unroll];
  int zc = INT32_MIN;  // lane s < 16: zhi8[s] (page_slices)
#pragma unroll
  for (int s = 0; s < kSlices && kPerKey; ++s)
    if (lane == s) zc = a.st.zhi[s];
#pragma unroll
  for (int u = 0; u < kQ8Unroll; ++u) {
    const int j = q8_local<kWaves>(wave, u), p = po + pm * j;
    int ns;
    q8_slices<kPerKey>(a, zc, p, N, ns, pr[u].mask);
    pr[u].n0 = p * kPage;
    const Q8Ref ref = q8_ref(hot, h, ent[u], j < count);
    q8_load_k(hot, a, ref, ns, lane, pr[u]);
    q8_load_v(hot, ref, lane, pr[u]);
  }
#pragma unroll
  for (int u = 0; u < kQ8Unroll; ++u) ent[u] = dec_fetch_entry(row, ord, q8_local<kWaves>(wave, kQ8Unroll + u));

  // Q^T fragments: lane holds query head t; fragment m is slice 2g + m % 2 + 8 (m / 2)
  u32x4 Qf[4];
  {
    const int qh = h * a.group + min(t, a.group - 1);
    const bool valid = t < a.group && N > 0;
    const uint16_t* qrow = a.q + static_cast<int64_t>(b) * a.q_sb + static_cast<int64_t>(qh) * a.q_sh;
    if (a.layout == kLayoutHalfSplit) {
#pragma unroll
      for (int m = 0; m < 4; ++m) Qf[m] = load_slice(qrow, kLayoutHalfSplit, 2 * g + (m & 1) + 8 * (m >> 1));
    } else {
#pragma unroll
      for (int m = 0; m < 4; ++m) Qf[m] = load_slice(qrow, kLayoutSortedPair, 2 * g + (m & 1) + 8 * (m >> 1));
    }
    if (a.rope_cs != nullptr) {
      float cs[4][8];
#pragma unroll
      for (int m = 0; m < 4; ++m) load_cs4(a.rope_cs, max(N - 1, 0), slice_pair0(2 * g + (m & 1) + 8 * (m >> 1)), cs[m]);
#pragma unroll
      for (int m = 0; m < 4; ++m) Qf[m] = rope_slice(Qf[m], cs[m]);
    }
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (!valid) Qf[m] = u32x4{0u, 0u, 0u, 0u};
  }
  // per-key rule: the distance limits of the lane's slices
  int zl[4] = {0, 0, 0, 0};
#pragma unroll
  for (int m = 0; m < 4 && kPerKey; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (g == i) zl[m] = a.st.zhi[2 * i + (m & 1) + 8 * (m >> 1)];

  f32x4 O[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) O[e] = f32x4{};
  float m_run = NEG_INF, l_run = 0.f;

  for (int i0 = 0; q8_local<kWaves>(wave, i0) < count; i0 += kQ8Unroll) {
#pragma unroll
    for (int u = 0; u < kQ8Unroll; ++u) {
      if (q8_local<kWaves>(wave, i0 + u) >= count) break;
      Q8Page& r = pr[u];
      if (kPerKey && r.mask) {
        const int age = (N - 1) - (r.n0 + t);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          if (age > zl[m]) {
            r.k[m >> 1][2 * (m & 1)] = 0u;
            r.k[m >> 1][2 * (m & 1) + 1] = 0u;
          }
      }
      const float sk = q8_scale<8>(r.e), sv = q8_scale<0>(r.e);
      f32x4 S = f32x4{};
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const u32x2 lo = q8_bf16(r.k[m >> 1][2 * (m & 1)], sk), hi = q8_bf16(r.k[m >> 1][2 * (m & 1) + 1], sk);
        S = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], hi[0], hi[1]}),
                                                    __builtin_bit_cast(bf16x8, Qf[m]), S, 0, 0, 0);
      }
      // S lane layout: query head t, tokens 4g + i
      const int tok0 = r.n0 + 4 * g;
      const bool tail = r.n0 + kPage > N;
      const int jn = q8_local<kWaves>(wave, i0 + kQ8Unroll + u);
      const bool reload = jn < count;
      bool mask_n = false;
      Q8Ref ref_n{0, false};
      if (reload) {
        int ns;
        q8_slices<kPerKey>(a, zc, po + pm * jn, N, ns, mask_n);
        ref_n = q8_ref(hot, h, ent[u], true);
        q8_load_k(hot, a, ref_n, ns, lane, r);
      }
      float mx = NEG_INF;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (tail && tok0 + i >= N) S[i] = NEG_INF;
        mx = fmaxf(mx, S[i]);
      }
      if (tail) {  // V codes of tokens past N to zero, so that 0 * V stays 0
        const int live = max(0, min(N - tok0, 4));
        const uint32_t keep = live == 4 ? 0xffffffffu : (1u << (8 * live)) - 1u;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int d = 0; d < 4; ++d) r.v[j][d] &= keep;
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
      for (int e = 0; e < 8; ++e)
        O[e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, q8_bf16(r.v[e >> 2][e & 3], sv)), pb,
                                                         O[e], 0, 0, 0);
      if (reload) {
        q8_load_v(hot, ref_n, lane, r);
        r.n0 = (po + pm * jn) * kPage;
        r.mask = mask_n;
        ent[u] = dec_fetch_entry(row, ord, q8_local<kWaves>(wave, i0 + 2 * kQ8Unroll + u));
      }
    }
  }

  const float l_tot = quad_sum(l_run);
  if (t < a.group) {
    // O[e][i]: dim 8 (4g + i) + e
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float* o = &sh_o[(out * kDecMaxGroup + t) * kD + 8 * (4 * g + i)];
      *reinterpret_cast<f32x4*>(o) = f32x4{O[0][i], O[1][i], O[2][i], O[3][i]};
      *reinterpret_cast<f32x4*>(o + 4) = f32x4{O[4][i], O[5][i], O[6][i], O[7][i]};
    }
    if (lane < 16) {
      sh_m[out * kDecMaxGroup + t] = m_run;
      sh_l[out * kDecMaxGroup + t] = l_tot;
    }
  }
}

template <int kWaves>
__device__ __forceinline__ void q8_first_entries(const int32_t* row, const PageOrder& ord, int wave, int max_pages,
                                                 int (&ent)[kQ8Unroll]) {
#pragma unroll
  for (int u = 0; u < kQ8Unroll; ++u) ent[u] = row[min(ord.po + ord.pm * q8_local<kWaves>(wave, u), max_pages - 1)];
}

template <bool kPerKey, int kWaves>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2)))
void decode_q8_kernel(const int32_t* page_table, const int32_t* seq_lens, const uint16_t* kv_cache, int max_pages,
                      int pages_per_split, int max_seq_len, int hkv, int num_pages, int n_splits, DecodeArgs a) {
  const DecHot hot{page_table, seq_lens, kv_cache, max_pages, pages_per_split, max_seq_len, hkv, num_pages, n_splits};
  __shared__ __attribute__((aligned(16))) float sh_o[kWaves * kDecMaxGroup * kD];
  __shared__ float sh_m[kWaves * kDecMaxGroup], sh_l[kWaves * kDecMaxGroup];
  const int s = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  PageOrder ord = page_order(s, n_splits, pages_per_split);
  int ent[kQ8Unroll];
  const int32_t* row = page_table + static_cast<int64_t>(b) * max_pages;
  q8_first_entries<kWaves>(row, ord, wave, max_pages, ent);
  const int N = max(0, min(seq_lens[b], max_seq_len));
  set_page_count(ord, s, n_splits, pages_per_split, (N + kPage - 1) / kPage);
  decode_pages_q8<kPerKey, kWaves>(hot, a, h, b, N, row, ord, wave, wave, ent, sh_o, sh_m, sh_l);
  __syncthreads();
  store_split<kWaves>(a, (static_cast<int64_t>(b) * hkv + h) * a.n_splits + s, h, b, sh_o, sh_m, sh_l);
}

// A workgroup per wave of a split, as decode_wave_kernel.
template <bool kPerKey>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2)))
void decode_q8_wave_kernel(const int32_t* page_table, const int32_t* seq_lens, const uint16_t* kv_cache, int max_pages,
                           int pages_per_split, int max_seq_len, int hkv, int num_pages, int n_splits, DecodeArgs a) {
  const DecHot hot{page_table, seq_lens, kv_cache, max_pages, pages_per_split, max_seq_len, hkv, num_pages, n_splits};
  const int s = blockIdx.x, h = blockIdx.y % hkv, wave = blockIdx.y / hkv;
  int b = blockIdx.z;
  if (a.by_length) b = a.batch <= 64 ? nth_longest<1>(seq_lens, a.batch, max_seq_len, b)
                                     : nth_longest<kDecSpreadBatch / 64>(seq_lens, a.batch, max_seq_len, b);
  PageOrder ord = page_order(s, n_splits, pages_per_split);
  int ent[kQ8Unroll];
  const int32_t* row = page_table + static_cast<int64_t>(b) * max_pages;
  q8_first_entries<kDecWaves>(row, ord, wave, max_pages, ent);
  const int N = max(0, min(seq_lens[b], max_seq_len));
  set_page_count(ord, s, n_splits, pages_per_split, (N + kPage - 1) / kPage);
  const int64_t unit = ((static_cast<int64_t>(b) * hkv + h) * n_splits + s) * kDecWaves + wave;
  float* ml = a.ws_ml + unit * 2 * a.group;
  decode_pages_q8<kPerKey, kDecWaves>(hot, a, h, b, N, row, ord, wave, 0, ent, a.ws_o + unit * a.group * kD, ml,
                                      ml + a.group);
}

hipError_t launch_decode_q8(const DecodeArgs& a, hipStream_t s) {
  if (a.batch <= 0) return hipSuccess;
#define ATF_Q8_LAUNCH(K, GRID, THREADS)                                                                              \
  hipLaunchKernelGGL(K, GRID, dim3(THREADS), 0, s, a.page_table, a.seq_lens, a.kv_cache, a.max_pages,                \
                     a.pages_per_split, a.max_seq_len, a.hkv, a.num_pages, a.n_splits, a)
  const dim3 grid(a.n_splits, a.hkv, a.batch), wgrid(a.n_splits, a.hkv * kDecWaves, a.batch);
  if (a.spread) {
    if (a.per_key) ATF_Q8_LAUNCH(decode_q8_wave_kernel<true>, wgrid, 64);
    else ATF_Q8_LAUNCH(decode_q8_wave_kernel<false>, wgrid, 64);
  } else if (a.waves == kDecWaves) {
    if (a.per_key) ATF_Q8_LAUNCH((decode_q8_kernel<true, kDecWaves>), grid, kDecWaves * 64);
    else ATF_Q8_LAUNCH((decode_q8_kernel<false, kDecWaves>), grid, kDecWaves * 64);
  } else {
    if (a.per_key) ATF_Q8_LAUNCH((decode_q8_kernel<true, kDecWavesShort>), grid, kDecWavesShort * 64);
    else ATF_Q8_LAUNCH((decode_q8_kernel<false, kDecWavesShort>), grid, kDecWavesShort * 64);
  }
#undef ATF_Q8_LAUNCH
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  return launch_decode_merge(a, s);
}

}  // namespace atf
