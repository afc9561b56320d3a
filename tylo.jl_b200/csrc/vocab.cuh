// What the scores and losses over a vocabulary share: one row of M logits x, read at temperature t.
//
//   y_j = (x_j - max x) / t,  L = sum exp(y_j),  p_j = exp(y_j) / L,  entropy = log L - sum exp(y_j) y_j / L
//
// Differences are taken before the scale: the lowest finite value overflows with a factor above 1, and a logit of a thousand
// would lose ten bits of its difference.  Both terms of the entropy are positive, so nothing cancels.
// Exponents are in units of log 2; the smallest that is used as a factor is kExpFloor, whose exp2 is zero: an entry of -Inf
// adds 0 * kExpFloor = 0 where 0 * -Inf would be NaN.  The sum itself takes the exponent as it is, so a NaN or +Inf reaches it.
// A row made only of -Inf has L = 0 and no probability anywhere.
#pragma once
#include "rowwise.cuh"

namespace tylo {

constexpr float kVocabLog2e = 1.4426950408889634f, kVocabLn2 = 0.6931471805599453f;
constexpr float kExpFloor = -160.f;

__device__ __forceinline__ float vocab_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row that may start and end inside a 16-byte packet: `head` elements before the first whole packet, `whole` packets,
// `tail` elements behind the last.  The at most 2 * (kVec - 1) single elements are dealt to the first threads, one each.
template <typename T> struct VocabRow {
  static constexpr int kVec = Elem<T>::kVec;
  int M, head, whole, tail;
  __device__ __forceinline__ VocabRow(const T* row, int m) : M(m) {
    head = min((int)(((16u - (unsigned)(reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / sizeof(T)), m);
    whole = (m - head) / kVec;
    tail = m - head - whole * kVec;
  }
  __device__ __forceinline__ int single(int tid) const {      // index of this thread's single element, -1: none
    return tid < head ? tid : (tid < head + tail ? M - tail + (tid - head) : -1);
  }
  __device__ __forceinline__ int index(int packet) const { return head + packet * kVec; }
};

// The logits may be overwritten by their gradient in the same kernel, so they are not read through the read-only path.
__device__ __forceinline__ uint4 ld_logits(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// Running statistics of a row or of a part of it: maximum, sum of exp2((x - m) * scale), sum of the same times its exponent.
struct VocabStats {
  float m, s, a;
  __device__ __forceinline__ void raise(float to, float scale) {       // to >= m
    const float d = fmaxf((m - to) * scale, kExpFloor), e = vocab_ex2(d);
    a = e * fmaf(d, s, a);
    s *= e;
    m = to;
  }
  __device__ __forceinline__ void join(float m2, float s2, float a2, float scale) {
    VocabStats o{m2, s2, a2};
    const float mn = fmaxf(m, o.m);
    raise(mn, scale);
    o.raise(mn, scale);
    s += o.s;
    a += o.a;
  }
};

// All threads receive the statistics of the CTA.  `scratch`: 96 floats, free again after the call.
template <int THREADS>
__device__ __forceinline__ void vocab_reduce(VocabStats& st, float scale, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    st.join(__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.a, o), scale);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) { scratch[warp] = st.m; scratch[32 + warp] = st.s; scratch[64 + warp] = st.a; }
  __syncthreads();
  const bool live = lane < THREADS / 32;
  st = {live ? scratch[lane] : -INFINITY, live ? scratch[32 + lane] : 0.f, live ? scratch[64 + lane] : 0.f};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    st.join(__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.a, o), scale);
  __syncthreads();
}

// Order of the alternatives as whole numbers: larger logits first, the lower index first among equals, a NaN above everything.
// Zero stands for "no entry" (no logit maps to it).
__device__ __forceinline__ uint32_t vocab_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);            // -0 equals +0
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float vocab_unkey(uint32_t k) {
  return k == 0xffffffffu ? __uint_as_float(0x7fffffffu) : __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t vocab_key(float x, int index) {
  return ((uint64_t)vocab_key(x) << 32) | (uint32_t)(0x7fffffff - index);
}
__device__ __forceinline__ int vocab_key_index(uint64_t k) { return 0x7fffffff - (int)(uint32_t)k; }

// Statistics of a whole row by one CTA.
template <typename T, int THREADS, bool ENTROPY>
__device__ __forceinline__ VocabStats vocab_row_stats(const T* x, const VocabRow<T>& r, float scale, float* scratch) {
  constexpr int VEC = Elem<T>::kVec, U = 4;
  VocabStats st{-INFINITY, 0.f, 0.f};
  const int one = r.single(threadIdx.x);
  if (one >= 0) {                                   // (a NaN or +Inf gives a NaN sum here as well)
    const float f = Elem<T>::to_f(x[one]);
    st.m = fmaxf(st.m, f);
    st.s = vocab_ex2((f - (st.m == -INFINITY ? 0.f : st.m)) * scale);
  }
  const T* base = x + r.head;
  for (int v0 = threadIdx.x; v0 < r.whole; v0 += U * THREADS) {
    float f[U][VEC];
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Pack<T> p;
      const int v = v0 + u * THREADS;
      if (v < r.whole) {
        p.raw = ld_logits(base + (size_t)v * VEC);
        p.unpack(f[u]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[u][j] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) mx = fmaxf(mx, f[u][j]);
    }
    if (mx > st.m) st.raise(mx, scale);
    const float mo = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float y = (f[u][j] - mo) * scale, e = vocab_ex2(y);
        st.s += e;
        if constexpr (ENTROPY) st.a = fmaf(e, fmaxf(y, kExpFloor), st.a);
      }
  }
  vocab_reduce<THREADS>(st, scale, scratch);
  return st;
}

inline int32_t check_vocab(const char* who, const void* X, int64_t M, int64_t N, int64_t ldx, float temperature) {
  TYLO_REQUIRE(X, TYLO_ERR_INVALID_ARGUMENT, "%s: X must be non-null", who);
  TYLO_REQUIRE(M > 0 && N > 0, TYLO_ERR_INVALID_ARGUMENT, "%s: extents must be positive (M=%lld, N=%lld)", who, (long long)M,
               (long long)N);
  TYLO_REQUIRE(ldx >= M, TYLO_ERR_INVALID_ARGUMENT, "%s: ldx (%lld) must be at least M (%lld)", who, (long long)ldx, (long long)M);
  TYLO_REQUIRE(M < 0x7fff0000LL && N <= 0x0fffffffLL, TYLO_ERR_UNSUPPORTED, "%s: M above 2^31-2^16 or N above 2^28-1 is not supported", who);
  TYLO_REQUIRE(temperature > 0.f && temperature <= 3.0e38f && 1.f / temperature <= 1e30f, TYLO_ERR_INVALID_ARGUMENT,
               "%s: temperature must be positive and finite", who);
  TYLO_REQUIRE(aligned16(X), TYLO_ERR_MISALIGNED, "%s: X must be 16-byte aligned", who);
  return TYLO_OK;
}

}  // namespace tylo
