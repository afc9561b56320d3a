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
#include <cooperative_groups.h>

#include <type_traits>

#include "rowwise.cuh"

namespace cg = cooperative_groups;

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
  __device__ __forceinline__ void join(VocabStats o, float scale) {
    const float mn = fmaxf(m, o.m);
    raise(mn, scale);
    o.raise(mn, scale);
    s += o.s;
    a += o.a;
  }
};

__device__ __forceinline__ void vocab_warp_reduce(VocabStats& st, float scale) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    st.join({__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.a, o)}, scale);
}

// All threads receive the statistics of the CTA, or of the cluster's CTAs that share a row.  `scratch`: 100 floats.  A cluster's CTAs
// must not leave before all have come back from here (their shared memory is read): see cluster_done.
template <int THREADS>
__device__ __forceinline__ void vocab_reduce(VocabStats& st, float scale, float* scratch, int parts) {
  vocab_warp_reduce(st, scale);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) { scratch[warp] = st.m; scratch[32 + warp] = st.s; scratch[64 + warp] = st.a; }
  __syncthreads();
  const bool live = lane < THREADS / 32;
  st = {live ? scratch[lane] : -INFINITY, live ? scratch[32 + lane] : 0.f, live ? scratch[64 + lane] : 0.f};
  vocab_warp_reduce(st, scale);
  if (parts > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    if (threadIdx.x == 0) { scratch[96] = st.m; scratch[97] = st.s; scratch[98] = st.a; }
    cluster.sync();
    const float* peer = cluster.map_shared_rank(scratch, lane < parts ? lane : 0);
    st = lane < parts ? VocabStats{peer[96], peer[97], peer[98]} : VocabStats{-INFINITY, 0.f, 0.f};
    vocab_warp_reduce(st, scale);
  }
  __syncthreads();
}

__device__ __forceinline__ void cluster_done(int parts) {
  if (parts > 1) cg::this_cluster().sync();
}

// The part of a row that one CTA works on: packets [lo, hi); the single elements belong to part 0.
struct VocabPart {
  int part, lo, hi;
  __device__ __forceinline__ VocabPart(int part_, int parts, int whole) : part(part_) {
    const int per = (whole + parts - 1) / parts;
    lo = min(part * per, whole);
    hi = min(lo + per, whole);
  }
};

// Largest element of U packets, a NaN passed over; 16-bit types two at a time.
template <typename T, int U> __device__ __forceinline__ float packets_max(const Pack<T> (&p)[U]) {
  if constexpr (sizeof(T) == 4) {
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(p[u].raw.x), __uint_as_float(p[u].raw.y)),
                         fmaxf(__uint_as_float(p[u].raw.z), __uint_as_float(p[u].raw.w))));
    return m;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    auto two = [](uint32_t w) { return *reinterpret_cast<const T2*>(&w); };
    T2 m = two(p[0].raw.x);
#pragma unroll
    for (int u = 0; u < U; ++u) m = __hmax2(m, __hmax2(__hmax2(two(p[u].raw.x), two(p[u].raw.y)), __hmax2(two(p[u].raw.z), two(p[u].raw.w))));
    const float r = fmaxf(Elem<T>::to_f(m.x), Elem<T>::to_f(m.y));
    return r == r ? r : -INFINITY;
  }
}

// -Inf in every element.
template <typename T> __device__ __forceinline__ uint4 no_logits() {
  const uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  return make_uint4(w, w, w, w);
}

// One thread's share of a part: every THREADS-th packet, U at a time with the next U on their way, and a single element.  The
// exponentials of a step are taken against the thread's own running maximum; sums are kept in two chains (packed fp32 pairs).
template <typename T, int THREADS, int U, bool ENTROPY>
__device__ __forceinline__ VocabStats vocab_thread_stats(const T* x, const VocabRow<T>& r, const VocabPart& part, float scale) {
  constexpr int VEC = Elem<T>::kVec;
  float m = -INFINITY;
  float2 s = make_float2(0.f, 0.f), a = s;
  const int one = part.part == 0 ? r.single(threadIdx.x) : -1;
  if (one >= 0) {                                   // (a NaN or +Inf gives a NaN sum here as below)
    const float f = Elem<T>::to_f(x[one]);
    m = fmaxf(m, f);
    s.x = vocab_ex2((f - (m == -INFINITY ? 0.f : m)) * scale);
  }
  const T* base = x + r.head;
  auto load = [&](Pack<T> (&p)[U], int v0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + u * THREADS;
      p[u].raw = v < part.hi ? ld_logits(base + (size_t)v * VEC) : no_logits<T>();
    }
  };
  auto take = [&](const Pack<T> (&p)[U]) {
    const float mx = packets_max<T, U>(p);
    if (mx > m) {
      const float d = fmaxf((m - mx) * scale, kExpFloor), e = vocab_ex2(d);
      if constexpr (ENTROPY) a = __fmul2_rn(make_float2(e, e), __ffma2_rn(make_float2(d, d), s, a));
      s = __fmul2_rn(make_float2(e, e), s);
      m = mx;
    }
    const float mo = m == -INFINITY ? 0.f : -m;
    const float2 nm = make_float2(mo, mo), sc = make_float2(scale, scale);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[VEC];
      p[u].unpack(f);
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        const float2 y = __fmul2_rn(__fadd2_rn(make_float2(f[j], f[j + 1]), nm), sc);
        const float2 e = make_float2(vocab_ex2(y.x), vocab_ex2(y.y));
        s = __fadd2_rn(s, e);
        if constexpr (ENTROPY) a = __ffma2_rn(e, make_float2(fmaxf(y.x, kExpFloor), fmaxf(y.y, kExpFloor)), a);
      }
    }
  };
  int v0 = part.lo + threadIdx.x;
  if (v0 < part.hi) {
    Pack<T> p[U], q[U];
    load(p, v0);
    while (true) {
      v0 += U * THREADS;
      if (v0 >= part.hi) { take(p); break; }
      load(q, v0);
      take(p);
      v0 += U * THREADS;
      if (v0 >= part.hi) { take(q); break; }
      load(p, v0);
      take(q);
    }
  }
  return {m, s.x + s.y, a.x + a.y};
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
