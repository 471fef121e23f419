// Writer of the paged cache of 8-bit floats, and its expansion into bf16 pages.
//
// Mathematics.  Per (page of 16 tokens, kv head, half): top = max |x| over the half's
// values, K rotated in fp32 first; e = the smallest integer with top <= 448 2^e, from
// the bits of top; code = e4m3(x 2^-e), round to nearest even, one rounding from the
// fp32 value (2^-4 of it at most, or 2^(e-10) below the smallest normal code).  The
// rotation's products and sums are rounded one by one (no fused multiply-add), so that
// the codes are those of the same expression elsewhere bit for bit.
//   A call that starts inside a page keeps the tokens before it: their exponent is the
// least that the page may have, and where the new one is larger their codes are
// shifted to it.  A call that writes a page's first slot begins the page anew.  Slots
// behind the call's last token become zero.  Infinities and NaN become the NaN code
// and count for no exponent.
//   Bound by HBM on long calls: K and V read once as bf16 (2 bytes an element), codes
// written once (1 byte), a (cos, sin) row of 512 bytes a position.  3 sequences of 20000
// tokens, 8 heads, 380 MB: 83 us, 4.6 TB/s, where a large copy reaches 4.7.  One token of
// each of 32 sequences: 5.1 us, a chain of four round trips (start, page entry and rows,
// the old codes, the store).
#include "atf_launch.h"

namespace atf {

constexpr float kQ8Max = 448.f;
constexpr uint32_t kInfBits = 0x7f800000u;

// The exponent of a half whose largest finite magnitude has these bits.
__device__ __forceinline__ int q8_exponent(uint32_t top) {
  // 448 2^e = 1.75 2^(e + 8): with top = 1.f 2^E, e = E - 8 where 1.f <= 1.75, else E - 7
  const int e = static_cast<int>(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kQ8MinExp), kQ8MaxExp);  // (top 0 or subnormal: the least)
}
__device__ __forceinline__ float exp2_int(int e) {  // -126 <= e <= 127
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Eight values times `inv` as codes.  odd: some value of the page is not finite, or
// the exponent was cut at its limit.
__device__ __forceinline__ u32x2 q8_codes(const float (&x)[8], float inv, bool odd) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = x[i] * inv;
  if (odd) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y[i] = (__float_as_uint(x[i]) & 0x7fffffffu) >= kInfBits ? __uint_as_float(0x7fc00000u)
                                                                : fminf(fmaxf(y[i], -kQ8Max), kQ8Max);
  }
  u32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
    w[i] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], p, true));
  }
  return w;
}

// Four codes of a half moved up by d exponents (scale = 2^-d).
__device__ __forceinline__ uint32_t q8_shift(uint32_t w, float scale) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, false);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, true);
  const int p = __builtin_amdgcn_cvt_pk_fp8_f32(a[0], a[1], 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(b[0], b[1], p, true));
}
__device__ __forceinline__ float shift_scale(int from, int to) { return exp2_int(max(from - to, -126)); }

// Bits of |x| for the page's maximum; a value that is not finite counts for nothing and is noted.
__device__ __forceinline__ void note(float x, uint32_t& top, uint32_t& odd) {
  const uint32_t m = __float_as_uint(x) & 0x7fffffffu;
  odd |= m >= kInfBits ? 1u : 0u;
  top = max(top, m >= kInfBits ? 0u : m);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) x = max(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), m)));
  return x;
}

// 4 x 4 bytes transposed: word i of the result holds byte i of the four words.
__device__ __forceinline__ u32x4 transpose4(const u32x4& w) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  return u32x4{__builtin_amdgcn_perm(b, a, 0x05040100u), __builtin_amdgcn_perm(b, a, 0x07060302u),
               __builtin_amdgcn_perm(d, c, 0x05040100u), __builtin_amdgcn_perm(d, c, 0x07060302u)};
}

// One workgroup of 128 threads per (page, kv head, sequence).
//   K: thread (level l = tid / 16, slot tid % 16) takes its token's level, rotates it and
// writes its 16 codes, the 16 bytes of the block at 16 tid.
//   V: thread tid takes 8 dims of tokens tid / 16 and 8 + tid / 16 (16 lanes read a whole
// row), their codes go to LDS by token, and thread (j, g, r) = tid takes a 4 x 4 square
// of it (dims 8r + 4j .. + 3, tokens 4g .. + 3), transposes it and writes the 16 bytes at
// 16 tid.
// grid: x = pages (from the call's first) and kv heads, y = sequence.  Workgroups go to the
// XCDs in turn: a page's heads lie on one XCD, one after the other, so that its (cos,
// sin) rows, as many bytes as a head's keys and values, come from that XCD's L2 (3 x 20000
// tokens of 8 heads 83.0 us, 89.9 with the heads last in the grid and the loads where their
// values are used).
__global__ __launch_bounds__(128) void kv_write_q8_kernel(KvWriteArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t sv[kPage][kD];
  __shared__ uint32_t s_top[2][2], s_odd[2];
  const int b = blockIdx.y, tid = threadIdx.x;
  const int j8 = blockIdx.x / a.page_round, turn = j8 / a.hkv, h = j8 - turn * a.hkv;
  const int start = a.start_pos[b];
  const KvRows rows = a.cu_tokens != nullptr ? kv_rows<true>(a, b) : kv_rows<false>(a, b);
  const int64_t end64 = static_cast<int64_t>(start) + rows.count;
  const int pidx = (max(start, 0) >> 4) + turn * a.page_round + (static_cast<int>(blockIdx.x) - j8 * a.page_round);
  const int64_t p0 = static_cast<int64_t>(pidx) * kPage;
  if (pidx >= a.max_pages || p0 >= end64) return;
  const int64_t lo = max(p0, static_cast<int64_t>(max(start, 0)));
  int64_t hi = min(p0 + kPage, end64);
  if (a.rope_cs != nullptr) hi = min(hi, static_cast<int64_t>(a.rope_max_pos));
  if (lo >= hi) return;
  const int s0 = static_cast<int>(lo - p0), s1 = static_cast<int>(hi - p0);
  const int pg = a.page_table[static_cast<int64_t>(b) * a.max_pages + pidx];  // waited for behind the rows' loads
  const int64_t row0 = rows.first + (p0 - start);  // source row of slot 0

  // Every load first (slots outside the call read a row of it, in bounds), then the
  // arithmetic: one memory round trip for all of them.
  const int l = tid >> 4, slot = tid & 15;
  const bool k_on = slot >= s0 && slot < s1;
  const int c0 = level_chunk0(a.layout, l);
  const uint16_t* krow = a.k_src + static_cast<int64_t>(b) * a.ks_b + (row0 + min(max(slot, s0), s1 - 1)) * a.ks_t +
                         static_cast<int64_t>(h) * a.ks_h;
  const u32x4 xk1 = ldg16(krow + c0), xk2 = ldg16(krow + level_chunk1(a.layout, l));
  u32x4 xv[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    xv[i] = ldg16(a.v_src + static_cast<int64_t>(b) * a.vs_b + (row0 + min(max(8 * i + l, s0), s1 - 1)) * a.vs_t +
                  static_cast<int64_t>(h) * a.vs_h + 8 * slot);
  float cs[16];
  if (a.rope_cs != nullptr) load_cs8(a.rope_cs, static_cast<int>(p0) + min(max(slot, s0), s1 - 1), c0, cs);
  if (pg < 0 || pg >= a.num_pages) return;
  const size_t blk = static_cast<size_t>(pg) * a.hkv + h;
  uint8_t* codes = reinterpret_cast<uint8_t*>(a.kv_cache) + blk * kQ8BlockBytes;
  // what the page keeps: the codes of slots before s0, under their exponents
  u32x4 old_k = {0u, 0u, 0u, 0u}, old_v = {0u, 0u, 0u, 0u};
  int ev = kQ8MinExp, ek = kQ8MinExp;
  if (s0 > 0) {
    old_v = ldg16(codes + 16 * tid);
    old_k = ldg16(codes + kQ8HalfBytes + 16 * tid);
    ev = a.kv_exps[2 * blk];
    ek = a.kv_exps[2 * blk + 1];
  }
  float ka[8] = {}, kb[8] = {};  // the level's two slices
  uint32_t k_top = 0, v_top = 0, odd = 0;
  if (k_on) {
    float x1[8], x2[8];
    unpack8(xk1, x1);
    unpack8(xk2, x2);
    if (a.rope_cs != nullptr) {
#pragma clang fp contract(off)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float c = cs[2 * i], s = cs[2 * i + 1], u = x1[i], w = x2[i];
        x1[i] = u * c - w * s;
        x2[i] = w * c + u * s;
      }
    }
    const bool hs = a.layout == kLayoutHalfSplit;  // (the slices of a level: kv_write_kernel)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ka[i] = hs ? x1[4 + i] : x1[i];
      ka[4 + i] = hs ? x2[4 + i] : x1[4 + i];
      kb[i] = hs ? x1[i] : x2[i];
      kb[4 + i] = hs ? x2[i] : x2[4 + i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      note(ka[i], k_top, odd);
      note(kb[i], k_top, odd);
    }
  }
  float v[2][8] = {};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int tok = 8 * i + l;
    if (tok >= s0 && tok < s1) {
      unpack8(xv[i], v[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) note(v[i][j], v_top, odd);
    }
  }
  const int wave = tid >> 6;
  k_top = wave_max(k_top);
  v_top = wave_max(v_top);
  odd = wave_max(odd);
  if ((tid & 63) == 0) {
    s_top[0][wave] = v_top;
    s_top[1][wave] = k_top;
    s_odd[wave] = odd;
  }
  __syncthreads();
  const int ev_n = max(ev, q8_exponent(max(s_top[0][0], s_top[0][1])));
  const int ek_n = max(ek, q8_exponent(max(s_top[1][0], s_top[1][1])));
  const bool plain = (s_odd[0] | s_odd[1]) == 0 && ev_n < kQ8MaxExp && ek_n < kQ8MaxExp;

  const float k_inv = exp2_int(-ek_n), v_inv = exp2_int(-ev_n);
  {
    u32x4 w = {0u, 0u, 0u, 0u};
    if (k_on) {
      const u32x2 wa = q8_codes(ka, k_inv, !plain), wb = q8_codes(kb, k_inv, !plain);
      w = u32x4{wa[0], wa[1], wb[0], wb[1]};
    } else if (slot < s0) {
      w = old_k;
      if (ek_n > ek) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = q8_shift(old_k[i], shift_scale(ek, ek_n));
      }
    }
    *reinterpret_cast<u32x4*>(codes + kQ8HalfBytes + 16 * tid) = w;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)  // (zeros for tokens the call does not cover)
    *reinterpret_cast<u32x2*>(&sv[8 * i + (tid >> 4)][8 * (tid & 15)]) = q8_codes(v[i], v_inv, !plain);
  __syncthreads();
  {
    const int j = tid >> 6, g = (tid >> 4) & 3, r = tid & 15;
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint32_t*>(&sv[4 * g + i][8 * r + 4 * j]);
    w = transpose4(w);
    const int kept = min(max(s0 - 4 * g, 0), 4);  // of the square's four tokens
    if (kept > 0) {
      const uint32_t keep = kept == 4 ? 0xffffffffu : (1u << (8 * kept)) - 1u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t o = ev_n > ev ? q8_shift(old_v[i], shift_scale(ev, ev_n)) : old_v[i];
        w[i] = (w[i] & ~keep) | (o & keep);
      }
    }
    *reinterpret_cast<u32x4*>(codes + 16 * tid) = w;
  }
  if (tid == 0) {
    a.kv_exps[2 * blk] = static_cast<int8_t>(ev_n);
    a.kv_exps[2 * blk + 1] = static_cast<int8_t>(ek_n);
  }
}

hipError_t launch_kv_write_q8(const KvWriteArgs& a, hipStream_t s) {
  if (a.n_tokens <= 0 || a.batch <= 0) return hipSuccess;
  // a call of n tokens touches at most ceil(n / 16) + 1 pages per sequence
  const int pages = (a.n_tokens + kPage - 1) / kPage + 1;
  KvWriteArgs k = a;
  k.page_round = pages < 8 ? pages : 8;
  const int64_t blocks = static_cast<int64_t>(pages + k.page_round - 1) / k.page_round * k.page_round * a.hkv;
  if (blocks > INT32_MAX) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(kv_write_q8_kernel, dim3(blocks, a.batch), dim3(128), 0, s, k);
  return hipGetLastError();
}

// A page of the 8-bit cache as a bf16 page: every code times its power of two, exact.
// One workgroup of 128 threads per (page-table entry, kv head); the thread takes the 16
// bytes of each half at 16 tid.  12 KB moved a (page, head), a copy's work: the prefill
// behind it grows with the queries, this does not.
//   Without an out_table a page goes to the block of its own number, whichever entries
// name it (several write the same bytes).
__global__ __launch_bounds__(128) void kv_expand_q8_kernel(KvExpandArgs a) {
  const int p = blockIdx.x, b = blockIdx.y, h = blockIdx.z, tid = threadIdx.x;
  const int64_t entry = static_cast<int64_t>(b) * a.n_pages + p;
  const bool held = a.seq_lens == nullptr || static_cast<int64_t>(p) * kPage < a.seq_lens[b];
  const int pg = held ? a.page_table[static_cast<int64_t>(b) * a.max_pages + p] : -1;
  const bool ok = pg >= 0 && pg < a.num_pages;
  const bool own = a.out_table == nullptr;
  if (!own && h == 0 && tid == 0) a.out_table[entry] = ok ? static_cast<int32_t>(entry) : -1;
  if (!ok) return;
  const size_t blk = static_cast<size_t>(pg) * a.hkv + h;
  const uint8_t* codes = a.codes + blk * kQ8BlockBytes;
  const u32x4 wv = ldg16(codes + 16 * tid), wk = ldg16(codes + kQ8HalfBytes + 16 * tid);
  const float sv = exp2_int(a.exps[2 * blk]), sk = exp2_int(a.exps[2 * blk + 1]);
  uint16_t* out = a.out + (static_cast<size_t>(own ? pg : entry) * a.hkv + h) * kKvBlockElems;
  auto pair = [](uint32_t w, float s) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true))};
  };
  const int l = tid >> 4, slot = tid & 15;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x2 x = pair(wk[2 * i], sk), y = pair(wk[2 * i + 1], sk);
    *reinterpret_cast<u32x4*>(out + kKHalfElems + (2 * l + i) * (kPage * kSliceDims) + slot * kSliceDims) =
        u32x4{x[0], x[1], y[0], y[1]};
  }
  const int j = tid >> 6, g = (tid >> 4) & 3, r = tid & 15;
#pragma unroll
  for (int d = 0; d < 4; ++d)
    *reinterpret_cast<u32x2*>(out + (8 * r + 4 * j + d) * kPage + v_slot(4 * g)) = pair(wv[d], sv);
}

hipError_t launch_kv_expand_q8(const KvExpandArgs& a, hipStream_t s) {
  if (a.batch <= 0 || a.n_pages <= 0) return hipSuccess;
  hipLaunchKernelGGL(kv_expand_q8_kernel, dim3(a.n_pages, a.batch, a.hkv), dim3(128), 0, s, a);
  return hipGetLastError();
}

}  // namespace atf
