// Log probabilities of given tokens, the entropy and the likeliest tokens of rows of logits.
//
// Mathematics.  One pass over a row x of V logits, in fp32 and powers of two: with u_i =
// (x_i - m) log2 e, m a logit, every thread keeps s = sum 2^u and t = sum u 2^u.  m is a wave's:
// its largest so far, give or take kSlack; when it is raised by d powers of two, s and t become
// s f and f (t - s d), f = 2^-d.  Then
//   log p(i) = x_i - m - log s,   entropy = (log2 s - t / s) / log2 e.
//   Logits of -inf count for nothing (0 in s and t); a row of nothing else has log
// probabilities of -inf and entropy 0.  NaN and +inf make the row's numbers NaN.
//   The likeliest tokens in the same pass.  A logit and its place make one number of 64
// bits, ordered as (value, lowest place first).  A wave keeps the best of what it has seen in
// LDS and gives the others its q-th best, q = ceil(top / 4): each of the 4 waves has q that
// reach the least of these, so that it is a bound, and 16 bytes of logits are looked at
// closer only if their largest reaches it.  For the first chunk the q-th best of a
// wave's lanes (each lane's largest) serve.
//   Bound by HBM on many rows (every logit is read once), with many alternatives by the vector
// units: 2048 rows of 152064 bf16 logits (normal, deviation 2) 118 us without alternatives (5.3 TB/s), 119
// with one, 135 with 20, 177 with 64; of fp32 logits 228 and, with 20, 248.  Some hundred rows are
// further from it (300 with 20 38 us, floor 17): whole chunks divide them unevenly.  What it came from, us
// for bf16 with none, 1 and 20: a workgroup of 512 that put its candidates in order together after
// every chunk, every element pushed by itself, one alternative 490; waves by themselves, the
// bound of all of them 136, 164, 195; joined by one wave, the row's filler left out 117, 137, 187;
// lanes' candidates side by side, ordered once 118, 135, 147; workgroups of 256 (four a CU, so that
// one's end runs beside the others' loads) 116, 130, 139.  One row takes 3.6 + 2.8 us of the two
// kernels, with five alternatives 8 + 4.3: a chain of loads, sums and LDS.
//   Requesting a chunk while the one before is summed changed nothing (130 without alternatives,
// 164 with one, before and after) and took 32 registers.
#include <type_traits>

#include "atf_launch.h"

namespace atf {

constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / 64;
constexpr int kLpRoom = 256;    // candidates of a wave (kTopMax and a push of 64 fit twice)
constexpr int kLpMerge = 2048;  // of a row's splits
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_inff();
constexpr float kLowest = -3.402823466e+38f;
constexpr float kSlack = 0.7f;  // a wave's m is raised for logits so far above it (2^u: 2 at most)

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
// bits, NaN of any kind as -inf.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return x == x ? k : 0x007fffffu;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
__device__ __forceinline__ uint64_t entry_of(float x, uint32_t at) {
  return (static_cast<uint64_t>(order_key(x)) << 32) | (0xffffffffu - at);
}
__device__ __forceinline__ uint64_t lane64(uint64_t x, int lane) {  // of a lane that is the same for the wave
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(x), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(x >> 32), lane);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
__device__ __forceinline__ uint64_t max64(uint64_t x, uint64_t y) { return x > y ? x : y; }
__device__ __forceinline__ uint64_t min64(uint64_t x, uint64_t y) { return x < y ? x : y; }

// Exchanges within rows of 16 lanes: with each in turn, lanes 0, 16, 32 and 48 get all of their rows.
constexpr int kLane1 = 0xb1, kLane2 = 0x4e, kMirror8 = 0x141, kMirror16 = 0x140;  // lane ^ 1, ^ 2, mirrored in 8, in 16
template <int kHow>
__device__ __forceinline__ uint32_t moved(uint32_t x) {
  return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), kHow, 0xf, 0xf, true));
}
template <int kHow>
__device__ __forceinline__ float moved(float x) {
  return __uint_as_float(moved<kHow>(__float_as_uint(x)));
}
__device__ __forceinline__ float lane_of(float x, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane));
}
// The largest of the wave's lanes, in every lane (unsigned 32 bits): maxima over rows of 16
// lanes, then over the rows.
__device__ __forceinline__ uint32_t wave_max32(uint32_t x) {
  x = max(x, moved<kLane1>(x));
  x = max(x, moved<kLane2>(x));
  x = max(x, moved<kMirror8>(x));
  x = max(x, moved<kMirror16>(x));
  const uint32_t a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16);
  const uint32_t c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
  return max(max(a, b), max(c, d));
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t x) {
  const uint32_t hi = wave_max32(static_cast<uint32_t>(x >> 32));
  const uint32_t lo = wave_max32(static_cast<uint32_t>(x >> 32) == hi ? static_cast<uint32_t>(x) : 0u);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
// The n-th largest of the lanes' numbers (different ones but for zeros), 0 if there are fewer.
__device__ __forceinline__ uint64_t wave_nth64(uint64_t x, int n) {
  if (n <= 8) {
    uint64_t y = 0;
    for (int i = 0; i < n; ++i) {
      y = wave_max64(x);
      x = x == y ? 0 : x;
    }
    return y;
  }
  int above = 0;
#pragma unroll 8
  for (int l = 0; l < 64; ++l) above += lane64(x, l) > x ? 1 : 0;
  const uint64_t at = __builtin_amdgcn_ballot_w64(above == n - 1 && x != 0);
  return at != 0 ? lane64(x, __builtin_ctzll(at)) : 0;
}
// The largest of three, not NaN if one is not, unless there is a signalling NaN among them: that
// makes it NaN.  (For fmaxf the compiler quiets the first pair of a chain and takes the others as they are.)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// A signalling NaN as a quiet one, all else as it is.  (Logits of bf16 and fp32 are taken bit by bit; those
// of fp16 come quiet from their conversion.)
__device__ __forceinline__ float quiet(float a) {
  float r;
  asm("v_max_f32 %0, %1, %1" : "=v"(r) : "v"(a));
  return r;
}
// LDS that only one wave uses: its accesses before and after keep their order.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// s and t relative to m (-inf: nothing yet).
struct LpStats {
  float m, s, t;
};
// The same sums relative to a larger m.
__device__ __forceinline__ void lp_raise(LpStats& a, float m) {
  const float d = (m - a.m) * kLog2e, f = __builtin_amdgcn_exp2f(-d);
  if (a.s != 0.f) {
    a.t = f == 0.f ? 0.f : f * __builtin_fmaf(a.s, -d, a.t);  // (s d may pass fp32 where nothing is left of it)
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
// log p of a logit x
__device__ __forceinline__ float lp_of(const LpStats& a, float log2_s, float x) {
  return x == kNegInf && a.s == a.s ? kNegInf : __builtin_fmaf(-log2_s, kLn2, x - a.m);
}
template <int kHow>
__device__ __forceinline__ void lp_join_moved(LpStats& a) {
  lp_join(a, LpStats{moved<kHow>(a.m), moved<kHow>(a.s), moved<kHow>(a.t)});
}
__device__ __forceinline__ float wave_sum(float x) {
  x += moved<kLane1>(x);
  x += moved<kLane2>(x);
  x += moved<kMirror8>(x);
  x += moved<kMirror16>(x);
  return (lane_of(x, 0) + lane_of(x, 16)) + (lane_of(x, 32) + lane_of(x, 48));
}

// The `top` best of n entries of `buf`, best first, to `out`; every thread of the workgroup.
__device__ __forceinline__ void rank_entries(const uint64_t* buf, int n, int top, uint64_t* out, int threads) {
  for (int i = threadIdx.x; i < n; i += threads) {
    const uint64_t x = buf[i];
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) above += buf[j] > x ? 1 : 0;
    if (above < top) out[above] = x;
  }
}

// What a wave has found: `len` entries in LDS, its `top` best among them.  Nothing below
// `floor` is among the row's best.
struct LpList {
  uint64_t* buf;    // [kLpRoom]
  uint64_t* given;  // [kLpWaves] each wave's q-th best (a wave with q = 0 gives none)
  unsigned long long* shared;  // the largest floor that a wave has found
  int len, top, q;
  uint64_t floor;
  int ordered;  // of the entries: as many as were there when they were last put in order
};
// The least of what the waves have given (it only grows): lane w looks at wave w's.
__device__ __forceinline__ uint64_t lp_least(const uint64_t* given) {
  static_assert(kLpWaves == 4, "two exchanges");
  uint64_t x = __hip_atomic_load(given + (threadIdx.x & (kLpWaves - 1)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  auto other = [&](uint32_t hi, uint32_t lo) { x = min64(x, (static_cast<uint64_t>(hi) << 32) | lo); };
  other(moved<kLane1>(static_cast<uint32_t>(x >> 32)), moved<kLane1>(static_cast<uint32_t>(x)));
  other(moved<kLane2>(static_cast<uint32_t>(x >> 32)), moved<kLane2>(static_cast<uint32_t>(x)));
  return lane64(x, 0);
}
// Only the `top` best are kept, best first.
__device__ __forceinline__ void lp_prune(LpList& a) {
  const int lane = threadIdx.x & 63;
  if (a.len == a.ordered) return;
  wave_fence();
  if (a.len <= 64) {
    const uint64_t x = lane < a.len ? a.buf[lane] : 0;
    int above = 0;
    for (int j = 0; j < a.len; ++j) above += lane64(x, j) > x ? 1 : 0;
    if (lane < a.len && above < a.top) a.buf[above] = x;
  } else {
    uint64_t x[kLpRoom / 64];
    int above[kLpRoom / 64];
#pragma unroll
    for (int i = 0; i < kLpRoom / 64; ++i) {
      x[i] = 64 * i + lane < a.len ? a.buf[64 * i + lane] : 0;
      above[i] = 0;
    }
    for (int j = 0; j < a.len; ++j) {
      const uint64_t y = a.buf[j];
#pragma unroll
      for (int i = 0; i < kLpRoom / 64; ++i) above[i] += y > x[i] ? 1 : 0;
    }
    wave_fence();
#pragma unroll
    for (int i = 0; i < kLpRoom / 64; ++i)
      if (64 * i + lane < a.len && above[i] < a.top) a.buf[above[i]] = x[i];
  }
  wave_fence();
  a.ordered = a.len = min(a.len, a.top);
  if (a.q > 0 && a.len >= a.q) {
    if (lane == 0) __hip_atomic_store(a.given + (threadIdx.x >> 6), a.buf[a.q - 1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    wave_fence();
    a.floor = max64(a.floor, lp_least(a.given));
  }
  if (a.len == a.top) a.floor = max64(a.floor, lane64(a.buf[a.top - 1], 0));  // one wave's `top` best are as good a bound
  if (lane == 0) atomicMax(a.shared, a.floor);
}
// The lanes' entries that reach the floor (0: none) into the list.
__device__ __forceinline__ void lp_push(LpList& a, uint64_t y) {
  uint64_t mask = __builtin_amdgcn_ballot_w64(y != 0 && y >= a.floor);
  if (a.len + __builtin_popcountll(mask) > kLpRoom) {
    lp_prune(a);
    mask = __builtin_amdgcn_ballot_w64(y != 0 && y >= a.floor);
  }
  const int at = a.len + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                                   __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0u));
  if (y != 0 && y >= a.floor) a.buf[at] = y;
  a.len += __builtin_popcountll(mask);
}

// A given token and its logit.
struct LpToken {
  int64_t id;
  float x;
};
template <int kType>
__device__ __forceinline__ LpToken lp_token(const LogprobArgs& a, int row, const void* x, int i) {
  LpToken t{-1, 0.f};
  if (i < a.n_tokens) {
    t.id = a.tokens[static_cast<int64_t>(row) * a.n_tokens + i];
    if (t.id >= 0 && t.id < a.vocab) t.x = LogitVec<kType>::one(x, t.id);
  }
  return t;
}
// The outputs of a row from its sums and its list.  token: the thread's first, requested before.
template <int kType>
__device__ __forceinline__ void lp_write(const LogprobArgs& a, int row, const void* x, const LpStats& st,
                                         const uint64_t* list, int len, LpToken token, int threads) {
  const float log2_s = log2f(st.s);
  for (int i = threadIdx.x; i < a.n_tokens; i += threads) {
    if (i >= threads) token = lp_token<kType>(a, row, x, i);
    a.logprobs[static_cast<int64_t>(row) * a.n_tokens + i] =
        token.id < 0 ? 0.f : token.id >= a.vocab ? __uint_as_float(0x7fc00000u) : lp_of(st, log2_s, token.x);
  }
  if (threadIdx.x == 0) a.entropy[row] = st.s == 0.f ? 0.f : (log2_s - st.t / st.s) * kLn2;
  for (int i = threadIdx.x; i < a.top; i += threads) {
    const uint64_t e = i < len ? list[i] : 0;
    const int64_t at = static_cast<int64_t>(row) * a.top + i;
    a.top_ids[at] = 0xffffffffu - static_cast<uint32_t>(e);
    a.top_logprobs[at] = lp_of(st, log2_s, key_value(static_cast<uint32_t>(e >> 32)));
  }
}

// One workgroup of 256 threads per (row, split): chunks of kVecs vectors of 16 bytes a
// thread, split y takes chunks y, y + gridDim.y, ..  The waves go through them by
// themselves; they meet at the end.  The few logits before the row's first 16-byte
// boundary and behind its last are lanes of split 0's first wave.
template <int kType, int kVecs, bool kTop>
__global__ __launch_bounds__(kLpThreads, 4) void token_logprobs_kernel(LogprobArgs a) {
  using V = LogitVec<kType>;
  constexpr int kE = V::kE;
  __shared__ uint64_t s_buf[kTop ? kLpWaves : 1][kTop ? kLpRoom : 1], s_all[kTop ? kLpWaves * kTopMax : 1], s_list[kTopMax];
  __shared__ uint64_t s_given[kLpWaves];
  __shared__ unsigned long long s_floor;
  __shared__ int s_count;
  __shared__ LpStats s_stats[kLpWaves];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const char* x = static_cast<const char*>(a.logits) + static_cast<int64_t>(row) * a.stride * V::kBytes;
  const int head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / V::kBytes, a.vocab);
  const int n_vec = (a.vocab - head) / kE;       // whole vectors
  const int rest = a.vocab - head - n_vec * kE;  // logits behind them
  const char* x0 = x + head * V::kBytes;
  if (kTop) {
    if (tid == 0) {
      s_count = 0;
      s_floor = 0;
    }
    if (tid < kLpWaves) s_given[tid] = 0;
    __syncthreads();
  }
  LpToken token{-1, 0.f};
  if (gridDim.y == 1 && wave == 0) token = lp_token<kType>(a, row, x, lane);
  LpStats st{kNegInf, 0.f, 0.f};  // (m is the wave's)
  bool careful = false;           // the wave has seen logits of which (x - m) log2 e is -inf
  LpList list{s_buf[kTop ? wave : 0], s_given, &s_floor, 0, a.top, 0, 0, 0};
  if (blockIdx.y == 0 && wave == 0 && head + rest > 0) {
    const int i = lane < 32 ? lane : a.vocab - rest + lane - 32;
    const bool on = lane < 32 ? lane < head : lane - 32 < rest;
    const float y = on ? V::one(x, i) : kNegInf;
    st.m = key_value(wave_max32(order_key(y)));
    const float u = (y - st.m) * kLog2e;
    st.s = y == kNegInf ? 0.f : __builtin_amdgcn_exp2f(u);
    st.t = st.s == 0.f ? 0.f : st.s * u;
    if (kTop) lp_push(list, on ? entry_of(y, i) : 0);
  }
  constexpr int kChunk = kLpThreads * kVecs;
  auto load = [&](int c0, u32x4 (&to)[kVecs]) {
    if (c0 + kChunk <= n_vec) {
#pragma unroll
      for (int k = 0; k < kVecs; ++k) to[k] = ldg16(x0 + 16 * static_cast<uint32_t>(c0 + k * kLpThreads + tid));
    } else {
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        const int j = c0 + k * kLpThreads + tid;
        to[k] = ldg16(x0 + 16 * static_cast<uint32_t>(min(j, n_vec - 1)));
        if (j >= n_vec) to[k] = u32x4{V::kFill, V::kFill, V::kFill, V::kFill};
      }
    }
  };
  for (int c0 = blockIdx.y * kChunk; c0 < n_vec; c0 += gridDim.y * kChunk) {
    u32x4 v[kVecs];
    load(c0, v);
    float vm[kVecs];  // the vectors' largest
    // The chunk's sums, a vector at a time.  The short way has a NaN in t where 2^u is 0 and u
    // -inf (masked logits), and where a logit is NaN: the chunk is then done again with u held above
    // -inf, and the largest taken past signalling NaN, and so are those after it.
    auto sums = [&](auto hold) {
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        float y[kE];
#pragma unroll
        for (int e = 0; e < kE; ++e) y[e] = V::get(v[k], e);
        vm[k] = max3(y[0], y[1], y[kE - 1]);
#pragma unroll
        for (int e = 2; e < kE - 1; e += 2) vm[k] = max3(vm[k], y[e], y[e + 1]);
        if (__builtin_amdgcn_ballot_w64(vm[k] > st.m + kSlack) != 0) lp_raise(st, key_value(wave_max32(order_key(vm[k]))));
        const float m = st.m == kNegInf ? 0.f : st.m;
        if (c0 + k * kLpThreads + tid < n_vec) {
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            const float u = (y[e] - m) * kLog2e, p = __builtin_amdgcn_exp2f(u);
            st.s += p;
            st.t = __builtin_fmaf(p, decltype(hold)::value ? fmaxf(u, kLowest) : u, st.t);
          }
        }
        if constexpr (decltype(hold)::value && kTop && kType != kLogitsFp16) {
          if (__builtin_amdgcn_ballot_w64(st.s != st.s) != 0) {  // a NaN, here or before: past a signalling one
            vm[k] = max3(quiet(y[0]), quiet(y[1]), quiet(y[kE - 1]));
#pragma unroll
            for (int e = 2; e < kE - 1; e += 2) vm[k] = max3(vm[k], quiet(y[e]), quiet(y[e + 1]));
          }
        }
      }
    };
    if (!careful) {
      const LpStats before = st;
      sums(std::false_type{});
      if (__builtin_amdgcn_ballot_w64(st.t != st.t) != 0) {
        careful = true;
        st = before;
      }
    }
    if (careful) sums(std::true_type{});
    float cm = vm[0];
#pragma unroll
    for (int k = 1; k < kVecs; ++k) cm = fmaxf(cm, vm[k]);
    if constexpr (kTop) {
      // a lane's best: the first place of its largest (a NaN at the front counts as -inf), 0 without one
      auto lane_best = [&] {
        int at = 0;
        u32x4 w = v[0];
#pragma unroll
        for (int k = kVecs - 1; k >= 0; --k) {
          if (vm[k] == cm) {
            at = k;
            w = v[k];
          }
        }
        int el = 0;
#pragma unroll
        for (int e = kE - 1; e >= 0; --e) el = V::get(w, e) == cm ? e : el;
        const int j = c0 + at * kLpThreads + tid;
        return j < n_vec ? entry_of(cm, head + j * kE + el) : 0;
      };
      // The first chunk's bounds, from the waves whose lanes all have logits.
      const int full = c0 == static_cast<int>(blockIdx.y) * kChunk ? min(kLpWaves, (n_vec - c0) / 64) : 0;
      if (full > 0) {  // (uniform)
        if (wave < full) {
          list.q = (a.top + full - 1) / full;
          const uint64_t nth = wave_nth64(lane_best(), list.q);
          if (lane == 0) s_given[wave] = nth;
          if (a.top == 1 && lane == 0) atomicMax(&s_floor, nth);
        } else if (lane == 0) {
          s_given[wave] = ~0ull;
        }
        __syncthreads();
        list.floor = max64(list.floor, lp_least(s_given));
      }
      list.floor = max64(list.floor, lane64(__hip_atomic_load(&s_floor, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP), 0));
      // what a logit has to reach: the floor's value, or the next one where all that is equal lies behind its place
      auto bar_of = [&] {
        const uint32_t key = static_cast<uint32_t>(list.floor >> 32), place = 0xffffffffu - static_cast<uint32_t>(list.floor);
        return list.floor == 0 ? kNegInf : key_value(key + (place < static_cast<uint32_t>(head + c0 * kE) ? 1u : 0u));
      };
      float bar = bar_of();
      const int over = __builtin_popcountll(__builtin_amdgcn_ballot_w64(!(cm < bar)));
      if (over != 0) {
        if (over >= 2 * a.top || over > 32) {  // many: the top-th best of the lanes is a better floor
          const uint64_t nth = wave_nth64(lane_best(), a.top);
          list.floor = max64(list.floor, nth);
          bar = bar_of();
        }
        // every lane takes its first vector with a candidate, of that the first candidate, then the
        // next, until no lane has one left
        uint32_t vectors = 0;
#pragma unroll
        for (int k = 0; k < kVecs; ++k)
          vectors |= !(vm[k] < bar) && c0 + k * kLpThreads + tid < n_vec ? 1u << k : 0u;
        while (__builtin_amdgcn_ballot_w64(vectors != 0) != 0) {
          const int k = vectors != 0 ? __builtin_ctz(vectors) : 0;
          u32x4 w = v[0];
#pragma unroll
          for (int i = 1; i < kVecs; ++i) w = k == i ? v[i] : w;
          uint32_t some = 0;
#pragma unroll
          for (int e = 0; e < kE; ++e) some |= V::get(w, e) < bar ? 0u : 1u << e;
          if (vectors == 0) some = 0;
          vectors &= vectors - 1;
          const int at = head + (c0 + k * kLpThreads + tid) * kE;
          while (__builtin_amdgcn_ballot_w64(some != 0) != 0) {
            const int e = some != 0 ? __builtin_ctz(some) : 0;
            float y = V::get(w, 0);
#pragma unroll
            for (int i = 1; i < kE; ++i) y = e == i ? V::get(w, i) : y;
            lp_push(list, some != 0 ? entry_of(y, at + e) : 0);
            some &= some - 1;
          }
        }
        if (full > 0 && c0 + static_cast<int>(gridDim.y) * kChunk < n_vec) lp_prune(list);  // (later chunks add little: what they do is put in order when the room ends)
      }
    }
  }
  // (the list of one chunk is short, and what the waves' lists hold is put in order below)
  if constexpr (kTop) {
    if (list.len > 64 || static_cast<int>(blockIdx.y + gridDim.y) * kChunk < n_vec) lp_prune(list);
  }
  st.s = wave_sum(st.s);
  st.t = wave_sum(st.t);
  if (lane == 0) s_stats[wave] = st;
  __syncthreads();
  int len = 0;
  if constexpr (kTop) {
    if (lane < list.len && list.buf[lane] >= max64(list.floor, s_floor)) s_all[atomicAdd(&s_count, 1)] = list.buf[lane];
    __syncthreads();
    len = min(s_count, a.top);
    rank_entries(s_all, s_count, a.top, s_list, kLpThreads);
    __syncthreads();
  }
  if (wave > 0) return;
  st = s_stats[lane & (kLpWaves - 1)];
  lp_join_moved<kLane1>(st);
  lp_join_moved<kLane2>(st);
  if (gridDim.y == 1) {
    lp_write<kType>(a, row, x, st, s_list, len, token, 64);
    return;
  }
  const int64_t part = static_cast<int64_t>(row) * gridDim.y + blockIdx.y;
  if (tid == 0) *reinterpret_cast<f32x4*>(a.ws_stats + 4 * part) = f32x4{st.m, st.s, st.t, 0.f};
  if (tid < a.top) a.ws_top[part * a.top + tid] = tid < len ? s_list[tid] : 0;
}

// The splits of a row joined: one workgroup a row.
constexpr int kLpMergeThreads = 256;
template <int kType>
__global__ __launch_bounds__(kLpMergeThreads) void logprobs_merge_kernel(LogprobArgs a) {
  __shared__ uint64_t buf[kLpMerge], list[kTopMax];
  __shared__ int s_count;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int64_t part = static_cast<int64_t>(row) * a.splits;
  const char* x = static_cast<const char*>(a.logits) + static_cast<int64_t>(row) * a.stride * LogitVec<kType>::kBytes;
  const LpToken token = lp_token<kType>(a, row, x, tid);
  if (tid == 0) s_count = 0;
  const int n = a.splits * a.top;
  constexpr int kMine = kLpMerge / kLpMergeThreads;
  uint64_t mine[kMine];
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int i = k * kLpMergeThreads + tid;
    mine[k] = i < n ? a.ws_top[part * a.top + i] : 0;
  }
  // A bound: of every list each step-th entry, a lane each (every wave the same), the n-th largest of them
  // with n step >= top.  So many entries reach it, and besides them fewer than `step` of each list
  // (n is 4 at most: finding it takes as long as a few more entries).  The least of the lists'
  // q-th best, q = ceil(top / lists), is a bound too, but one that a short last list spoils: 48 rows
  // with 64 alternatives 34 us for both kernels, 20 with this.  With more lists than lanes a lane takes the largest of several lists' first, and the largest of the lists' last serves too.
  const int step = a.splits > 64 ? 1 : max((a.top * a.splits + 63) / 64, (a.top + 3) / 4);
  const int each = a.splits > 64 ? 1 : a.top / max(step, 1);
  uint64_t some = 0, last = 0;
  if (a.top > 0) {
    for (int i = lane; i < a.splits * each; i += 64) {
      some = max64(some, a.ws_top[(part + i / each) * a.top + (i % each + 1) * step - 1]);
      if (a.splits > 64) last = max64(last, a.ws_top[(part + i) * a.top + a.top - 1]);
    }
  }
  LpStats st{kNegInf, 0.f, 0.f};
  for (int i = lane; i < a.splits; i += 64) {
    const f32x4 p = *reinterpret_cast<const f32x4*>(a.ws_stats + 4 * (part + i));
    lp_join(st, LpStats{p[0], p[1], p[2]});
  }
  lp_join_moved<kLane1>(st);
  lp_join_moved<kLane2>(st);
  lp_join_moved<kMirror8>(st);
  lp_join_moved<kMirror16>(st);
  auto row16 = [&](int l) { return LpStats{lane_of(st.m, l), lane_of(st.s, l), lane_of(st.t, l)}; };
  LpStats joined = row16(0), far = row16(32);
  lp_join(joined, row16(16));
  lp_join(far, row16(48));
  lp_join(joined, far);
  int len = 0;
  if (a.top > 0) {
    uint64_t bound = wave_nth64(some, (a.top + step - 1) / step);
    if (a.splits > 64) bound = max64(bound, wave_max64(last));
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kMine; ++k)
      if (mine[k] != 0 && mine[k] >= bound) buf[atomicAdd(&s_count, 1)] = mine[k];
    __syncthreads();
    len = min(s_count, a.top);
    rank_entries(buf, s_count, a.top, list, kLpMergeThreads);
    __syncthreads();
  }
  lp_write<kType>(a, row, x, joined, list, len, token, kLpMergeThreads);
}

// Vectors of a thread's chunk, with alternatives and without: with them the chunks are few (each
// begins with a look at the others' bounds), without them more waves fit (2048 x 152064 bf16 with
// 20 alternatives 147 us at 8 and 161 at 4 in workgroups of 512; without 118 and 115).
constexpr int kLpVecsTop = 8, kLpVecsSums = 4;

// Workgroups of a row: four a CU for all rows together, a chunk each at least, and no more than
// the merge has room for.  Chunks of 8 KB instead of 32 KB for the splits were slower with
// alternatives, whose first chunk costs the most (300 x 152064 bf16 with 20: 53 us, 37 with 32 KB).
int logprob_splits(int rows, int vocab, int type, int top) {
  const int64_t bytes = static_cast<int64_t>(vocab) * (type == kLogitsFp32 ? 4 : 2);
  const int64_t chunk = 16 * kLpThreads * (top > 0 ? kLpVecsTop : kLpVecsSums);
  int64_t n = (bytes + chunk - 1) / chunk;
  if (rows > 0 && n > 1024 / rows) n = 1024 / rows;
  if (top > 0 && n > kLpMerge / top) n = kLpMerge / top;
  return n < 1 ? 1 : static_cast<int>(n);
}

template <int kType>
static void launch_logprobs(const LogprobArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(a.top > 0 ? (token_logprobs_kernel<kType, kLpVecsTop, true>) : (token_logprobs_kernel<kType, kLpVecsSums, false>),
                     dim3(a.rows, a.splits), dim3(kLpThreads), 0, s, a);
  if (a.splits > 1) hipLaunchKernelGGL(logprobs_merge_kernel<kType>, dim3(a.rows), dim3(kLpMergeThreads), 0, s, a);
}

hipError_t launch_token_logprobs(const LogprobArgs& a, hipStream_t s) {
  if (a.rows <= 0) return hipSuccess;
  if (a.type == kLogitsBf16) launch_logprobs<kLogitsBf16>(a, s);
  else if (a.type == kLogitsFp16) launch_logprobs<kLogitsFp16>(a, s);
  else launch_logprobs<kLogitsFp32>(a, s);
  return hipGetLastError();
}

}  // namespace atf
