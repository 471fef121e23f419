// Log probabilities of given tokens, the entropy and the likeliest tokens of rows of logits.
//
// Mathematics.  One pass over a row x of V logits keeps, for each thread, m = the largest
// so far, s = sum exp(x - m) and t = sum (x - m) exp(x - m), all fp32; two of them
// join as s = s1 f1 + s2 f2, t = f1 (t1 + s1 (m1 - m)) + .., f = exp(m_i - m).  Then
//   log p(i) = (x_i - m) - log s,   entropy = log s - t / s.
// Logits of -inf count for nothing (0 in s and t); a row of nothing else has log
// probabilities of -inf and entropy 0.  NaN and +inf make the row's numbers NaN.
//   The likeliest tokens in the same pass.  A logit and its place make one number of 64
// bits, ordered as (value, lowest place first).  A chunk of the row stays in registers;
// a wave takes the top-th largest of its lanes' best as a bound (so many are at least that
// good), the workgroup the best bound of its waves and of the list so far, and only
// what passes it, about `top` a row, goes through LDS to be ranked by counting.
//   Bound by HBM: every logit is read once.
#include "atf_launch.h"

namespace atf {

constexpr int kLpThreads = 512;
constexpr int kLpWaves = kLpThreads / 64;
constexpr int kLpRoom = 2048;  // candidates ranked at a time
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
constexpr float kLowest = -3.402823466e+38f;

template <int kType>
struct LogitVec {  // 16 bytes of logits
  static constexpr int kE = kType == kLogitsFp32 ? 4 : 8;
  static constexpr int kBytes = kType == kLogitsFp32 ? 4 : 2;
  static constexpr uint32_t kFill = kType == kLogitsBf16 ? 0xff80ff80u : kType == kLogitsFp16 ? 0xfc00fc00u : 0xff800000u;
  __device__ static float get(const u32x4& v, int e) {
    if constexpr (kType == kLogitsFp32) return __uint_as_float(v[e]);
    const uint32_t w = v[e >> 1];
    if constexpr (kType == kLogitsBf16) return __uint_as_float((e & 1) ? (w & 0xffff0000u) : (w << 16));
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>((e & 1) ? (w >> 16) : w)));
  }
  __device__ static float one(const void* row, int64_t i) {
    if constexpr (kType == kLogitsFp32) return static_cast<const float*>(row)[i];
    const uint16_t h = static_cast<const uint16_t*>(row)[i];
    if constexpr (kType == kLogitsBf16) return bf16_to_f32(h);
    return static_cast<float>(__builtin_bit_cast(_Float16, h));
  }
};

// A value as 32 bits that are ordered as the values are; equal values (0 and -0) the same
// bits, NaN below everything.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return x == x ? k : 0u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);  // (0: a NaN)
}
__device__ __forceinline__ uint64_t entry_of(float x, uint32_t at) {
  return (static_cast<uint64_t>(order_key(x)) << 32) | (0xffffffffu - at);
}
__device__ __forceinline__ uint64_t shfl64(uint64_t x, int lane) {
  const uint32_t lo = __shfl(static_cast<int>(x), lane), hi = __shfl(static_cast<int>(x >> 32), lane);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint32_t lo = __shfl_xor(static_cast<int>(x), m), hi = __shfl_xor(static_cast<int>(x >> 32), m);
    const uint64_t y = (static_cast<uint64_t>(hi) << 32) | lo;
    x = y > x ? y : x;
  }
  return x;
}

struct LpStats {
  float m, s, t;
};
// The same sums relative to a maximum that is no smaller.
__device__ __forceinline__ void lp_raise(LpStats& a, float m) {
  if (a.s != 0.f) {
    const float d = a.m - m, f = __builtin_amdgcn_exp2f(d * kLog2e);
    a.t = f == 0.f ? 0.f : f * __builtin_fmaf(a.s, d, a.t);  // (s d may pass fp32 where nothing is left of it)
    a.s *= f;
  }
  a.m = m;
}
__device__ __forceinline__ void lp_join(LpStats& a, LpStats b) {
  const float m = fmaxf(a.m, b.m);
  lp_raise(a, m);
  lp_raise(b, m);
  a.s += b.s;
  a.t += b.t;
}
__device__ __forceinline__ LpStats lp_wave(LpStats a) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) lp_join(a, LpStats{__shfl_xor(a.m, m), __shfl_xor(a.s, m), __shfl_xor(a.t, m)});
  return a;
}
// log p of a logit x
__device__ __forceinline__ float lp_of(const LpStats& a, float log_s, float x) {
  const float d = x - a.m;
  return x == kNegInf && a.s == a.s ? kNegInf : d - log_s;
}
// The `top` best of n entries of `buf`, best first, to `out`; every thread of the workgroup.
__device__ __forceinline__ void rank_entries(const uint64_t* buf, int n, int top, uint64_t* out, int threads) {
  for (int i = threadIdx.x; i < n; i += threads) {
    const uint64_t x = buf[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += buf[j] > x ? 1 : 0;
    if (above < top) out[above] = x;
  }
}

// The outputs of a row from its sums and its list.
template <int kType>
__device__ __forceinline__ void lp_write(const LogprobArgs& a, int row, const void* x, const LpStats& st,
                                         const uint64_t* list, int len, int threads) {
  const float log_s = logf(st.s);
  for (int i = threadIdx.x; i < a.n_tokens; i += threads) {
    const int64_t at = static_cast<int64_t>(row) * a.n_tokens + i;
    const int64_t tok = a.tokens[at];
    a.logprobs[at] = tok < 0 ? 0.f
                     : tok >= a.vocab ? __uint_as_float(0x7fc00000u)
                                      : lp_of(st, log_s, LogitVec<kType>::one(x, tok));
  }
  if (threadIdx.x == 0) a.entropy[row] = st.s == 0.f ? 0.f : log_s - st.t / st.s;
  for (int i = threadIdx.x; i < a.top; i += threads) {
    const uint64_t e = i < len ? list[i] : 0;
    const int64_t at = static_cast<int64_t>(row) * a.top + i;
    a.top_ids[at] = 0xffffffffu - static_cast<uint32_t>(e);
    a.top_logprobs[at] = lp_of(st, log_s, key_value(static_cast<uint32_t>(e >> 32)));
  }
}

// One workgroup of 512 threads per (row, split): chunks of kVecs vectors of 16 bytes a
// thread, split y takes chunks y, y + gridDim.y, ..  The few logits before the row's first
// 16-byte boundary and behind its last are two more vectors, read one by one.
template <int kType, int kVecs, bool kTop>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_kernel(LogprobArgs a) {
  using V = LogitVec<kType>;
  constexpr int kE = V::kE;
  __shared__ uint64_t buf[kTop ? kLpRoom : 1], list[kTopMax];
  __shared__ uint64_t s_bound, s_wave[kLpWaves];
  __shared__ int s_count;
  __shared__ LpStats s_stats[kLpWaves];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const char* x = static_cast<const char*>(a.logits) + static_cast<int64_t>(row) * a.stride * V::kBytes;
  const int head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / V::kBytes, a.vocab);
  const int n_vec = (a.vocab - head) / kE;            // whole vectors
  const int rest = a.vocab - head - n_vec * kE;       // logits behind them
  const int n_all = n_vec + (rest > 0 ? 1 : 0) + (head > 0 ? 1 : 0);
  const char* x0 = x + head * V::kBytes;
  // the place of element 0 of vector j: the vectors, the rest, the head (its last elements)
  auto place = [&](int j) {
    return j < n_vec ? head + j * kE : (j == n_vec && rest > 0) ? head + n_vec * kE : head - kE;
  };
  auto edge = [&](int j) {
    u32x4 v = {V::kFill, V::kFill, V::kFill, V::kFill};
    if (j < n_all) {
      const int at = place(j);
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const int i = at + e;
        if (i >= 0 && i < a.vocab && (j == n_vec && rest > 0 ? true : i < head)) {
          if constexpr (kType == kLogitsFp32) {
            v[e] = reinterpret_cast<const uint32_t*>(x)[i];
          } else {
            const uint32_t h = reinterpret_cast<const uint16_t*>(x)[i];
            v[e >> 1] = (e & 1) ? ((v[e >> 1] & 0x0000ffffu) | (h << 16)) : ((v[e >> 1] & 0xffff0000u) | h);
          }
        }
      }
    }
    return v;
  };
  // whether element e of vector j is a logit of the row
  auto real = [&](int j, int e) {
    const int i = place(j) + e;
    return j < n_vec || (j < n_all && i >= 0 && i < a.vocab && (j != n_vec || rest > 0 || i < head));
  };

  LpStats st{kNegInf, 0.f, 0.f};
  uint64_t bound = 0;  // of the list: nothing below it is among the best
  int len = 0;
  if (kTop && tid == 0) {
    s_count = 0;
    s_bound = 0;
  }
  if (kTop) __syncthreads();
  constexpr int kChunk = kLpThreads * kVecs;
  for (int c0 = blockIdx.y * kChunk; c0 < n_all; c0 += gridDim.y * kChunk) {
    u32x4 v[kVecs];
    if (c0 + kChunk <= n_vec) {
#pragma unroll
      for (int k = 0; k < kVecs; ++k) v[k] = ldg16(x0 + static_cast<int64_t>(c0 + k * kLpThreads + tid) * 16);
    } else {
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        const int j = c0 + k * kLpThreads + tid;
        v[k] = j < n_vec ? ldg16(x0 + static_cast<int64_t>(j) * 16) : edge(j);
      }
    }
    float cm = kNegInf;
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
#pragma unroll
      for (int e = 0; e < kE; ++e) cm = fmaxf(cm, V::get(v[k], e));
    if (cm > st.m) lp_raise(st, cm);
    const float m = st.m == kNegInf ? 0.f : st.m;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const float d = V::get(v[k], e) - m, p = __builtin_amdgcn_exp2f(d * kLog2e);
        st.s += p;
        st.t = __builtin_fmaf(p, fmaxf(d, kLowest), st.t);
      }
    }
    if constexpr (kTop) {
      const bool maybe = order_key(cm) >= static_cast<uint32_t>(bound >> 32);
      uint64_t best = 0, limit = bound;
      if (__builtin_amdgcn_ballot_w64(maybe) != 0) {
        if (maybe) {
#pragma unroll
          for (int k = 0; k < kVecs; ++k) {
            const int j = c0 + k * kLpThreads + tid;
#pragma unroll
            for (int e = 0; e < kE; ++e) {
              const uint64_t y = real(j, e) ? entry_of(V::get(v[k], e), place(j) + e) : 0;
              best = y > best ? y : best;
            }
          }
        }
        const uint64_t over = __builtin_amdgcn_ballot_w64(best > bound);
        if (__builtin_popcountll(over) >= a.top) {  // the top-th best lane: a bound
          int above = 0;
          for (int l = 0; l < 64; ++l) above += shfl64(best, l) > best ? 1 : 0;
          const uint64_t at = __builtin_amdgcn_ballot_w64(above == a.top - 1 && best > bound);
          if (at != 0) {
            limit = shfl64(best, __builtin_ctzll(at));
            if (lane == 0) atomicMax(reinterpret_cast<unsigned long long*>(&s_bound), limit);
          }
        }
      }
      __syncthreads();
      limit = s_bound > bound ? s_bound : bound;
      if (best >= limit && best > bound) {
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
          const int j = c0 + k * kLpThreads + tid;
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            const uint64_t y = real(j, e) ? entry_of(V::get(v[k], e), place(j) + e) : 0;
            if (y >= limit && y > bound) {
              const int at = len + atomicAdd(&s_count, 1);
              if (at < kLpRoom) buf[at] = y;
            }
          }
        }
      }
      __syncthreads();
      const int fresh = s_count;
      if (fresh > 0) {  // (uniform)
        int n = len + fresh;
        if (n <= kLpRoom) {
          rank_entries(buf, n, a.top, list, kLpThreads);
          n = min(n, a.top);
        } else {
          // More candidates than room (a thread's chunk holds many of the best): one by one.
          uint64_t last = ~0ull;
          for (n = 0; n < a.top; ++n) {
            uint64_t y = tid < len && buf[tid] < last ? buf[tid] : 0;
#pragma unroll
            for (int k = 0; k < kVecs; ++k) {
              const int j = c0 + k * kLpThreads + tid;
#pragma unroll
              for (int e = 0; e < kE; ++e) {
                const uint64_t z = real(j, e) ? entry_of(V::get(v[k], e), place(j) + e) : 0;
                y = z < last && z > y ? z : y;
              }
            }
            y = wave_max64(y);
            if (lane == 0) s_wave[wave] = y;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kLpWaves; ++w) y = s_wave[w] > y ? s_wave[w] : y;
            __syncthreads();
            if (y == 0) break;
            if (tid == 0) list[n] = y;
            last = y;
          }
        }
        __syncthreads();
        for (int i = tid; i < n; i += kLpThreads) buf[i] = list[i];
        len = n;
        bound = n == a.top ? list[n - 1] : 0;
        if (tid == 0) {
          s_count = 0;
          s_bound = bound;
        }
        __syncthreads();
      }
    }
  }
  st = lp_wave(st);
  if (lane == 0) s_stats[wave] = st;
  __syncthreads();
  st = s_stats[0];
#pragma unroll
  for (int w = 1; w < kLpWaves; ++w) lp_join(st, s_stats[w]);
  if (gridDim.y == 1) {
    lp_write<kType>(a, row, x, st, buf, len, kLpThreads);
    return;
  }
  const int64_t part = static_cast<int64_t>(row) * gridDim.y + blockIdx.y;
  if (tid == 0) *reinterpret_cast<f32x4*>(a.ws_stats + 4 * part) = f32x4{st.m, st.s, st.t, 0.f};
  if (tid < a.top) a.ws_top[part * a.top + tid] = tid < len ? buf[tid] : 0;
}

// The splits of a row joined: one workgroup a row.
constexpr int kLpMergeThreads = 256;
template <int kType>
__global__ __launch_bounds__(kLpMergeThreads) void logprobs_merge_kernel(LogprobArgs a) {
  __shared__ uint64_t buf[kLpRoom], list[kTopMax];
  __shared__ int s_count;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int64_t part = static_cast<int64_t>(row) * a.splits;
  if (tid == 0) s_count = 0;
  LpStats st{kNegInf, 0.f, 0.f};
  uint64_t bound = 0;  // the best of the splits' last: so many are at least that good
  for (int i = lane; i < a.splits; i += 64) {  // (every wave the same)
    const f32x4 p = *reinterpret_cast<const f32x4*>(a.ws_stats + 4 * (part + i));
    lp_join(st, LpStats{p[0], p[1], p[2]});
    if (a.top > 0) {
      const uint64_t y = a.ws_top[(part + i) * a.top + a.top - 1];
      bound = y > bound ? y : bound;
    }
  }
  st = lp_wave(st);
  bound = wave_max64(bound);
  __syncthreads();
  for (int i = tid; i < a.splits * a.top; i += kLpMergeThreads) {
    const uint64_t y = a.ws_top[part * a.top + i];
    if (y >= bound && y != 0) buf[atomicAdd(&s_count, 1)] = y;
  }
  __syncthreads();
  const int n = s_count;
  rank_entries(buf, n, a.top, list, kLpMergeThreads);
  __syncthreads();
  const char* x = static_cast<const char*>(a.logits) + static_cast<int64_t>(row) * a.stride * LogitVec<kType>::kBytes;
  lp_write<kType>(a, row, x, st, list, min(n, a.top), kLpMergeThreads);
}

constexpr int kLpVecs = 8, kLpVecsSplit = 2;  // vectors of a thread's chunk: rows whole, rows split

// Workgroups of a row: two a CU for all rows together, a chunk of 16 KB each at least, and no
// more than the merge has room for.
int logprob_splits(int rows, int vocab, int type, int top) {
  const int64_t bytes = static_cast<int64_t>(vocab) * (type == kLogitsFp32 ? 4 : 2);
  int64_t n = (bytes + 16 * kLpThreads * kLpVecsSplit - 1) / (16 * kLpThreads * kLpVecsSplit);
  if (rows > 0 && n > 512 / rows) n = 512 / rows;
  if (top > 0 && n > kLpRoom / top) n = kLpRoom / top;
  return n < 1 ? 1 : static_cast<int>(n);
}

template <int kType>
static void launch_logprobs(const LogprobArgs& a, hipStream_t s) {
  const dim3 grid(a.rows, a.splits), block(kLpThreads);
  if (a.splits == 1) {
    hipLaunchKernelGGL(a.top > 0 ? (token_logprobs_kernel<kType, kLpVecs, true>) : (token_logprobs_kernel<kType, kLpVecs, false>),
                       grid, block, 0, s, a);
  } else {
    hipLaunchKernelGGL(a.top > 0 ? (token_logprobs_kernel<kType, kLpVecsSplit, true>)
                                 : (token_logprobs_kernel<kType, kLpVecsSplit, false>),
                       grid, block, 0, s, a);
    hipLaunchKernelGGL(logprobs_merge_kernel<kType>, dim3(a.rows), dim3(kLpMergeThreads), 0, s, a);
  }
}

hipError_t launch_token_logprobs(const LogprobArgs& a, hipStream_t s) {
  if (a.rows <= 0) return hipSuccess;
  if (a.type == kLogitsBf16) launch_logprobs<kLogitsBf16>(a, s);
  else if (a.type == kLogitsFp16) launch_logprobs<kLogitsFp16>(a, s);
  else launch_logprobs<kLogitsFp32>(a, s);
  return hipGetLastError();
}

}  // namespace atf
