// RMS norm of each head's queries and keys with the rotation of their positions in the
// same pass, on rows and into the paged caches.
//
// Mathematics.  Per (token, head) row x of 128: y = x (mean(x^2) + eps)^-1/2 w, and for a
// token with a position z[r] = y[r] c_r - y[r + 64] s_r, z[r + 64] = y[r + 64] c_r + y[r] s_r.
// Everything is fp32 from the bf16 input to the one rounding of the result (bf16, or
// the 8-bit cache's code).
//   Eight lanes hold a row: lane i dims 8i .. 8i + 7 and the same + 64, so that a rotated
// pair lies in one lane, the sum of squares takes three lane exchanges, and the lane's
// 16 dims are a level of the cache's K half (level 7 - i).  Bound by HBM on long calls: a
// row read and written, a (cos, sin) row of 512 bytes a position.  37000 packed rows of 24 + 8
// heads, 613 MB: 117 us, 5.2 TB/s, as a large copy; into the bf16 cache 2 x 16000 tokens of 28 + 4
// heads with their values, 597 MB: 113 us, 5.3 TB/s; turns of 11 sequences into the 8-bit cache,
// 105 MB: 23 to 25 us.  A step's append of 32 tokens 3.7 us, two round trips before the stores, into the
// 8-bit cache 5.3 (in a graph, the bf16 cache's 3.0): a page's kernel for a token.
#include "atf_launch.h"
#include "atf_q8.h"

namespace atf {

// The sum over the 8 lanes of a row, the same bits in all of them.
__device__ __forceinline__ float sum8(float x) {
  auto add = [](float v, int moved) { return v + __int_as_float(moved); };
  x = add(x, __builtin_amdgcn_mov_dpp(__float_as_int(x), 0xb1, 0xf, 0xf, true));   // lane ^ 1
  x = add(x, __builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4e, 0xf, 0xf, true));   // lane ^ 2
  x = add(x, __builtin_amdgcn_mov_dpp(__float_as_int(x), 0x141, 0xf, 0xf, true));  // 7 - lane, of the eight
  return x;
}

// The lane's 16 weights (dims 8i .. 8i + 7, then the same + 64).
__device__ __forceinline__ void load_weights(const void* w, bool fp32, int i, float (&w1)[8], float (&w2)[8]) {
  if (fp32) {
    const float* p = static_cast<const float*>(w) + 8 * i;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const u32x4 a = ldg16(p + 4 * j), b = ldg16(p + kP + 4 * j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w1[4 * j + e] = __uint_as_float(a[e]);
        w2[4 * j + e] = __uint_as_float(b[e]);
      }
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(w) + 8 * i;
    unpack8(ldg16(p), w1);
    unpack8(ldg16(p + kP), w2);
  }
}

// Whether mean(x^2) + eps is a normal fp32 number.  A row of which it is not is scaled by a power of two and squared
// again (kAny): squares of large rows pass fp32, those of small ones are subnormal, which the root takes for 0.
// Scaling rounds nothing that a result shows, and a normal mean has lost less than 2^-26 of itself with the squares
// that are not normal.
__device__ __forceinline__ bool plain_mean(float m) {
  constexpr int kPositiveNormal = 0x100;
  return __builtin_amdgcn_classf(m, kPositiveNormal);
}

// A lane's 16 dims of a row (a: the first halves of its pairs, b: the second) normed and,
// with `rope`, rotated by its pairs' (cos, sin).  Returns plain_mean: without kAny the results of a
// row that is not are not its own.
template <bool kAny>
__device__ __forceinline__ bool norm_rotate(const u32x4& a, const u32x4& b, const float (&w1)[8], const float (&w2)[8],
                                            float eps, bool rope, const float (&cs)[16], float (&z1)[8],
                                            float (&z2)[8]) {
  float x1[8], x2[8];
  unpack8(a, x1);
  unpack8(b, x2);
  auto mean_of = [&](float e) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = __builtin_fmaf(x1[i], x1[i], s);
#pragma unroll
    for (int i = 0; i < 8; ++i) s = __builtin_fmaf(x2[i], x2[i], s);
    return __builtin_fmaf(sum8(s), 1.f / kD, e);
  };
  float m = mean_of(eps);
  const bool plain = plain_mean(m);
  if (kAny && __builtin_expect(__builtin_amdgcn_ballot_w64(!plain) != 0, 0)) {
    const float scale = plain ? 1.f : m < 1.f ? 0x1p100f : 0x1p-70f;  // (a row's eight lanes alike)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x1[i] *= scale;
      x2[i] *= scale;
    }
    m = mean_of(eps * scale * scale);
  }
  const float inv = __builtin_amdgcn_rsqf(m);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y1 = x1[i] * inv * w1[i], y2 = x2[i] * inv * w2[i];
    z1[i] = rope ? rope_first(y1, y2, cs[2 * i], cs[2 * i + 1]) : y1;
    z2[i] = rope ? rope_second(y1, y2, cs[2 * i], cs[2 * i + 1]) : y2;
  }
  return plain;
}

__device__ __forceinline__ void store_row(uint16_t* row, int i, const float (&z1)[8], const float (&z2)[8]) {
  *reinterpret_cast<u32x4*>(row + 8 * i) = pack8(z1);
  *reinterpret_cast<u32x4*>(row + kP + 8 * i) = pack8(z2);
}

// ---- rows ----

// A wave takes a token's heads, eight at a time (q's, then k's), the groups blockIdx.y,
// blockIdx.y + gridDim.y, ..: four workgroups' waves a (token, y).
constexpr int kNormWaves = 4;
__global__ __launch_bounds__(64 * kNormWaves) void qk_norm_rows_kernel(QkNormArgs a) {
  const int lane = threadIdx.x & 63, i = lane & 7;
  const int t = blockIdx.x * kNormWaves + (threadIdx.x >> 6);
  if (t >= a.rows) return;
  const bool rope = a.rope_cs != nullptr;
  float cs[16] = {};
  if (rope) {
    const int pos = a.positions[t];
    if (pos < 0 || pos >= a.rope_max_pos) return;
    load_cs8(a.rope_cs, pos, 8 * i, cs);
  }
  for (int h = 8 * blockIdx.y + (lane >> 3); h < a.hq + a.hk; h += 8 * gridDim.y) {
    const bool is_q = h < a.hq;
    const int hh = is_q ? h : h - a.hq;
    const uint16_t* x = is_q ? a.q + t * a.q_st + hh * a.q_sh : a.k + t * a.k_st + hh * a.k_sh;
    const u32x4 x1 = ldg16(x + 8 * i), x2 = ldg16(x + kP + 8 * i);
    float w1[8], w2[8], z1[8], z2[8];
    load_weights(is_q ? a.q_weight : a.k_weight, a.weights_fp32, i, w1, w2);
    norm_rotate<true>(x1, x2, w1, w2, a.eps, rope, cs, z1, z2);
    uint16_t* out = is_q ? a.q_out + (static_cast<int64_t>(t) * a.hq + hh) * kD
                         : a.k_out + (static_cast<int64_t>(t) * a.hk + hh) * kD;
    store_row(out, i, z1, z2);
  }
}

hipError_t launch_qk_norm_rows(const QkNormArgs& a, hipStream_t s) {
  const int heads = a.hq + a.hk;
  if (a.rows <= 0 || heads <= 0) return hipSuccess;
  const int groups = (heads + 7) / 8;
  hipLaunchKernelGGL(qk_norm_rows_kernel, dim3((a.rows + kNormWaves - 1) / kNormWaves, groups < 4 ? groups : 4),
                     dim3(64 * kNormWaves), 0, s, a);
  return hipGetLastError();
}

// ---- into the caches ----

// The slots of a page that a call covers: [s0, s1), and the source row of slot 0.
struct PageSpan {
  int s0, s1;
  int64_t row0;
};

// One workgroup of 128 threads per (page, unit, sequence): the units are the kv heads, then
// eight q heads at a time.  Lane 8j + i of wave w takes 16 dims of token 8w + j.
//   K: normed and rotated into the page's K half; V as it is (kv_write_kernel, and for
// the 8-bit cache kv_write_q8_kernel, have the halves' layouts and what a page that is
// covered in part keeps).  Q: to its rows of q_out.
// grid: x = pages (from the call's first) and units, the units of `page_round` pages in turn,
// so that a page's units run on one XCD (workgroups go to the XCDs in turn) and its (cos,
// sin) rows come from its L2; y = sequence.
constexpr int kNormQHeads = 8;  // q heads of a unit
template <bool kQ8>
__global__ __launch_bounds__(128) void qk_norm_write_kernel(QkNormArgs n) {
  const KvWriteArgs& a = n.kv;
  __shared__ __attribute__((aligned(16))) uint16_t sv[kPage][kD];  // V's rows, or their codes
  __shared__ uint32_t s_top[2][2], s_odd[2];
  const int b = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int units = a.hkv + (n.hq + kNormQHeads - 1) / kNormQHeads;
  const int j8 = blockIdx.x / a.page_round, turn = j8 / units, unit = j8 - turn * units;
  const int start = a.start_pos[b];
  const KvRows rows = kv_rows<true>(a, b);
  const int64_t end64 = static_cast<int64_t>(start) + rows.count;
  const int pidx = (max(start, 0) >> 4) + turn * a.page_round + (static_cast<int>(blockIdx.x) - j8 * a.page_round);
  const int64_t p0 = static_cast<int64_t>(pidx) * kPage;
  const bool rope = a.rope_cs != nullptr;
  const int64_t lo = max(p0, static_cast<int64_t>(max(start, 0)));
  int64_t hi = min(p0 + kPage, end64);
  if (rope) hi = min(hi, static_cast<int64_t>(a.rope_max_pos));
  if (lo >= hi) return;
  const PageSpan sp{static_cast<int>(lo - p0), static_cast<int>(hi - p0), rows.first + (p0 - start)};
  // (slots outside the call read a row of it, in bounds, and write nothing of it)
  const int i = lane & 7, slot = 8 * wave + (lane >> 3);
  const bool on = slot >= sp.s0 && slot < sp.s1;
  const int near = min(max(slot, sp.s0), sp.s1 - 1);
  const int64_t row = sp.row0 + near;
  float cs[16] = {}, w1[8], w2[8];
  if (rope) load_cs8(a.rope_cs, static_cast<int>(p0) + near, 8 * i, cs);

  if (unit >= a.hkv) {  // ---- Q ----
    load_weights(n.q_weight, n.weights_fp32, i, w1, w2);
    const int h0 = (unit - a.hkv) * kNormQHeads;
    const uint16_t* x = n.q + row * n.q_st;
    constexpr int kBatch = 4;  // heads whose loads are in flight together
#pragma unroll
    for (int j0 = 0; j0 < kNormQHeads; j0 += kBatch) {
      u32x4 x1[kBatch], x2[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int64_t at = min(h0 + j0 + j, n.hq - 1) * n.q_sh;
        x1[j] = ldg16(x + at + 8 * i);
        x2[j] = ldg16(x + at + kP + 8 * i);
      }
      // (rows that are not plain are done again behind the four: a branch after each head made 32 single
      // tokens into the 8-bit cache 0.2 us slower, this one 0)
      bool plain = true;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int h = h0 + j0 + j;
        float z1[8], z2[8];
        plain &= norm_rotate<false>(x1[j], x2[j], w1, w2, n.eps, rope, cs, z1, z2);
        if (on && h < n.hq) store_row(n.q_out + (row * n.hq + h) * kD, i, z1, z2);
      }
      if (__builtin_amdgcn_ballot_w64(!plain) != 0) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int h = h0 + j0 + j;
          float z1[8], z2[8];
          norm_rotate<true>(x1[j], x2[j], w1, w2, n.eps, rope, cs, z1, z2);
          if (on && h < n.hq) store_row(n.q_out + (row * n.hq + h) * kD, i, z1, z2);
        }
      }
    }
    return;
  }

  // ---- K and V of one head ----
  if (pidx >= a.max_pages) return;
  const int pg = a.page_table[static_cast<int64_t>(b) * a.max_pages + pidx];
  const uint16_t* krow = a.k_src + row * a.ks_t + static_cast<int64_t>(unit) * a.ks_h;
  const u32x4 xk1 = ldg16(krow + 8 * i), xk2 = ldg16(krow + kP + 8 * i);
  u32x4 xv[2];  // V: 8 dims of tokens tid / 16 and 8 + tid / 16
#pragma unroll
  for (int r = 0; r < 2; ++r)
    xv[r] = ldg16(a.v_src + (sp.row0 + min(max(8 * r + (tid >> 4), sp.s0), sp.s1 - 1)) * a.vs_t +
                  static_cast<int64_t>(unit) * a.vs_h + 8 * (tid & 15));
  load_weights(n.k_weight, n.weights_fp32, i, w1, w2);
  if (pg < 0 || pg >= a.num_pages) return;
  const size_t blk = static_cast<size_t>(pg) * a.hkv + unit;
  float z1[8], z2[8];
  norm_rotate<true>(xk1, xk2, w1, w2, n.eps, rope, cs, z1, z2);
  // the level's two slices: the upper four of its pairs (first halves, then second), the lower four
  const float ka[8] = {z1[4], z1[5], z1[6], z1[7], z2[4], z2[5], z2[6], z2[7]};
  const float kb[8] = {z1[0], z1[1], z1[2], z1[3], z2[0], z2[1], z2[2], z2[3]};
  const int l = kLevels - 1 - i;

  if constexpr (!kQ8) {
    uint16_t* page = a.kv_cache + blk * kKvBlockElems;
    if (on) {
      uint16_t* kdst = page + kKHalfElems + (2 * l) * (kPage * kSliceDims) + slot * kSliceDims;
      *reinterpret_cast<u32x4*>(kdst) = pack8(ka);
      *reinterpret_cast<u32x4*>(kdst + kPage * kSliceDims) = pack8(kb);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) *reinterpret_cast<u32x4*>(&sv[8 * r + (tid >> 4)][8 * (tid & 15)]) = xv[r];
    __syncthreads();
    uint16_t* vdst = page + tid * kPage;  // row tid of V^T
    uint32_t w[8] = {};
    if (sp.s0 > 0 || sp.s1 < kPage) {
      const u32x4 r0 = ldg16(vdst), r1 = ldg16(vdst + 8);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = r0[e];
        w[4 + e] = r1[e];
      }
    }
#pragma unroll
    for (int tok = 0; tok < kPage; ++tok) {
      if (tok >= sp.s0 && tok < sp.s1) {
        const int sl = v_slot(tok);
        const uint32_t val = sv[tok][tid];
        w[sl >> 1] = (sl & 1) ? ((w[sl >> 1] & 0x0000ffffu) | (val << 16)) : ((w[sl >> 1] & 0xffff0000u) | val);
      }
    }
    *reinterpret_cast<u32x4*>(vdst) = u32x4{w[0], w[1], w[2], w[3]};
    *reinterpret_cast<u32x4*>(vdst + 8) = u32x4{w[4], w[5], w[6], w[7]};
  } else {
    uint8_t* codes = reinterpret_cast<uint8_t*>(a.kv_cache) + blk * kQ8BlockBytes;
    const int k_at = kQ8HalfBytes + 16 * (kPage * l + slot);
    // what the page keeps: the codes of slots before s0, under their exponents
    u32x4 old_k = {0u, 0u, 0u, 0u}, old_v = {0u, 0u, 0u, 0u};
    int ev = kQ8MinExp, ek = kQ8MinExp;
    if (sp.s0 > 0) {
      old_v = ldg16(codes + 16 * tid);
      old_k = ldg16(codes + k_at);
      ev = a.kv_exps[2 * blk];
      ek = a.kv_exps[2 * blk + 1];
    }
    uint32_t k_top = 0, v_top = 0, odd = 0;
    if (on) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        note(ka[e], k_top, odd);
        note(kb[e], k_top, odd);
      }
    }
    float v[2][8] = {};
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int tok = 8 * r + (tid >> 4);
      if (tok >= sp.s0 && tok < sp.s1) {
        unpack8(xv[r], v[r]);
#pragma unroll
        for (int e = 0; e < 8; ++e) note(v[r][e], v_top, odd);
      }
    }
    k_top = wave_max(k_top);
    v_top = wave_max(v_top);
    odd = wave_max(odd);
    if (lane == 0) {
      s_top[0][wave] = v_top;
      s_top[1][wave] = k_top;
      s_odd[wave] = odd;
    }
    __syncthreads();
    const int ev_n = max(ev, q8_exponent(max(s_top[0][0], s_top[0][1])));
    const int ek_n = max(ek, q8_exponent(max(s_top[1][0], s_top[1][1])));
    const bool plain = (s_odd[0] | s_odd[1]) == 0 && ev_n < kQ8MaxExp && ek_n < kQ8MaxExp;
    u32x4 w = {0u, 0u, 0u, 0u};
    if (on) {
      const u32x2 wa = q8_codes(ka, exp2_int(-ek_n), !plain), wb = q8_codes(kb, exp2_int(-ek_n), !plain);
      w = u32x4{wa[0], wa[1], wb[0], wb[1]};
    } else if (slot < sp.s0) {
      w = old_k;
      if (ek_n > ek) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = q8_shift(old_k[e], shift_scale(ek, ek_n));
      }
    }
    *reinterpret_cast<u32x4*>(codes + k_at) = w;
    uint8_t* vb = reinterpret_cast<uint8_t*>(&sv[0][0]);  // [16 tokens][128]
#pragma unroll
    for (int r = 0; r < 2; ++r)  // (zeros for tokens the call does not cover)
      *reinterpret_cast<u32x2*>(vb + (8 * r + (tid >> 4)) * kD + 8 * (tid & 15)) = q8_codes(v[r], exp2_int(-ev_n), !plain);
    __syncthreads();
    const int j = tid >> 6, g = (tid >> 4) & 3, r = tid & 15;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = *reinterpret_cast<const uint32_t*>(vb + (4 * g + e) * kD + 8 * r + 4 * j);
    w = transpose4(w);
    const int kept = min(max(sp.s0 - 4 * g, 0), 4);  // of the square's four tokens
    if (kept > 0) {
      const uint32_t keep = kept == 4 ? 0xffffffffu : (1u << (8 * kept)) - 1u;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t o = ev_n > ev ? q8_shift(old_v[e], shift_scale(ev, ev_n)) : old_v[e];
        w[e] = (w[e] & ~keep) | (o & keep);
      }
    }
    *reinterpret_cast<u32x4*>(codes + 16 * tid) = w;
    if (tid == 0) {
      a.kv_exps[2 * blk] = static_cast<int8_t>(ev_n);
      a.kv_exps[2 * blk + 1] = static_cast<int8_t>(ek_n);
    }
  }
}

// A few tokens into the bf16 cache (a decode step's append): one wave per (eight heads, token,
// sequence), the heads q's, then k's, then v's.  V's elements go to their slots one by one, so
// nothing is read back or staged.  Same results, same skips.
// grid: x = heads in eights, y = token of the sequence, z = sequence.
constexpr int kNormAppendTokens = 4;
__global__ __launch_bounds__(64) void qk_norm_append_kernel(QkNormArgs n) {
  const KvWriteArgs& a = n.kv;
  const int lane = threadIdx.x, i = lane & 7, b = blockIdx.z, t = blockIdx.y;
  const int u = 8 * blockIdx.x + (lane >> 3);
  const KvRows rows = kv_rows<true>(a, b);
  if (t >= rows.count) return;
  const int64_t row = rows.first + t;
  const int kind = u < n.hq ? 0 : u < n.hq + a.hkv ? 1 : 2;  // q, k, v
  const int h = u - (kind == 0 ? 0 : kind == 1 ? n.hq : n.hq + a.hkv);
  const bool on = kind < 2 || h < a.hkv;
  const uint16_t* x = kind == 0 ? n.q + row * n.q_st + h * n.q_sh
                      : kind == 1 ? a.k_src + row * a.ks_t + h * a.ks_h
                                  : a.v_src + row * a.vs_t + min(h, a.hkv - 1) * a.vs_h;
  const u32x4 x1 = ldg16(x + 8 * i), x2 = ldg16(x + kP + 8 * i);
  float w1[8], w2[8];
  load_weights(kind == 0 ? n.q_weight : n.k_weight, n.weights_fp32, i, w1, w2);
  const bool rope = a.rope_cs != nullptr;
  const int64_t pos = static_cast<int64_t>(a.start_pos[b]) + t, pidx = pos >> 4;
  if (pos < 0 || (rope && pos >= a.rope_max_pos)) return;
  float cs[16] = {};
  if (rope) load_cs8(a.rope_cs, static_cast<int>(pos), 8 * i, cs);
  const int pg = pidx < a.max_pages ? a.page_table[static_cast<int64_t>(b) * a.max_pages + pidx] : -1;
  float z1[8], z2[8];
  norm_rotate<true>(x1, x2, w1, w2, n.eps, rope, cs, z1, z2);
  if (kind == 0) {
    store_row(n.q_out + (row * n.hq + h) * kD, i, z1, z2);
    return;
  }
  if (!on || pg < 0 || pg >= a.num_pages) return;
  uint16_t* page = a.kv_cache + (static_cast<size_t>(pg) * a.hkv + h) * kKvBlockElems;
  const int slot = static_cast<int>(pos) & (kPage - 1);
  if (kind == 1) {
    const float ka[8] = {z1[4], z1[5], z1[6], z1[7], z2[4], z2[5], z2[6], z2[7]};
    const float kb[8] = {z1[0], z1[1], z1[2], z1[3], z2[0], z2[1], z2[2], z2[3]};
    uint16_t* kdst = page + kKHalfElems + 2 * (kLevels - 1 - i) * (kPage * kSliceDims) + slot * kSliceDims;
    *reinterpret_cast<u32x4*>(kdst) = pack8(ka);
    *reinterpret_cast<u32x4*>(kdst + kPage * kSliceDims) = pack8(kb);
  } else {
    uint16_t* vdst = page + v_slot(slot);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      vdst[(8 * i + 2 * e) * kPage] = static_cast<uint16_t>(x1[e]);
      vdst[(8 * i + 2 * e + 1) * kPage] = static_cast<uint16_t>(x1[e] >> 16);
      vdst[(kP + 8 * i + 2 * e) * kPage] = static_cast<uint16_t>(x2[e]);
      vdst[(kP + 8 * i + 2 * e + 1) * kPage] = static_cast<uint16_t>(x2[e] >> 16);
    }
  }
}

hipError_t launch_qk_norm_write(const QkNormArgs& a, hipStream_t s) {
  if (a.kv.n_tokens <= 0 || a.kv.batch <= 0) return hipSuccess;
  if (a.kv.n_tokens <= kNormAppendTokens && a.kv.kv_exps == nullptr) {
    hipLaunchKernelGGL(qk_norm_append_kernel, dim3((a.hq + 2 * a.kv.hkv + 7) / 8, a.kv.n_tokens, a.kv.batch), dim3(64), 0, s, a);
    return hipGetLastError();
  }
  // a call of n tokens touches at most ceil(n / 16) + 1 pages per sequence
  const int pages = (a.kv.n_tokens + kPage - 1) / kPage + 1;
  QkNormArgs n = a;
  n.kv.page_round = pages < 8 ? pages : 8;
  const int64_t units = a.kv.hkv + (a.hq + kNormQHeads - 1) / kNormQHeads;
  const int64_t blocks = static_cast<int64_t>(pages + n.kv.page_round - 1) / n.kv.page_round * n.kv.page_round * units;
  if (blocks >= (int64_t(1) << 32) / 128) return hipErrorInvalidConfiguration;  // (2^32 threads)
  hipLaunchKernelGGL(a.kv.kv_exps != nullptr ? qk_norm_write_kernel<true> : qk_norm_write_kernel<false>,
                     dim3(blocks, a.kv.batch), dim3(128), 0, s, n);
  return hipGetLastError();
}

}  // namespace atf
