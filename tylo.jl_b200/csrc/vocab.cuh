// What the scores and losses over a vocabulary share: one row of M logits x, read at temperature t.
//
//   y_j = (x_j - max x) / t,  L = sum exp(y_j),  p_j = exp(y_j) / L,  entropy = log L - sum exp(y_j) y_j / L
//
// Differences are taken before the scale: the lowest finite value overflows with a factor above 1, and a logit of a thousand
// would lose ten bits of its difference.  Both terms of the entropy are positive, so it does not cancel.
// Exponents are in units of log 2; the smallest that is used as a factor is kExpFloor, whose exp2 is zero: an entry of -Inf
// adds 0 * kExpFloor = 0 where 0 * -Inf would be NaN.  The sum itself takes the exponent as it is, so a NaN or +Inf reaches it.
// A row made only of -Inf has L = 0 and no probability anywhere.
//
// What the kernels take now stands at the heads of logprob.cu and distill.cu.  The figures in the comments below, and beside single choices
// there, set two forms against each other at the time of the choice, in short runs: they hold as pairs.
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

// The same with a place in L2: a row that will be read again stays there before what is read or written once (4096 x 131072 bf16, value
// and gradient 414 us, 454 without), and is the first to go when it has been.  (A row that gets zeros is not read again: it stays until
// other rows push it out.)
__device__ __forceinline__ uint64_t keep_policy() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t drop_policy() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint4 ld_logits(const void* p, uint64_t policy) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.L2::cache_hint.v4.u32 {%0,%1,%2,%3}, [%4], %5;"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p), "l"(policy) : "memory");
  return v;
}

// Running statistics of a row or of a part of it: largest logit, the reference that the exponentials are taken against, sum of
// e = exp2((x - ref) * scale), sum of e times its exponent.  The reference follows the maximum only when that is more than
// kRefSlack (in units of log 2) above it: sums in floating point are as good (the entropy's second sum to kRefSlack * 2^-24), and the
// branch that rescales them stays rare (2048 x 131072 bf16 92 us with the maximum as reference, 89 so).
constexpr float kRefSlack = 8.f;

struct VocabStats {
  float m, ref, s, a;
  __device__ __forceinline__ void refer(float to, float scale) {
    const float d = fmaxf((ref - to) * scale, kExpFloor), e = vocab_ex2(d);
    a = e * fmaf(d, s, a);
    s *= e;
    ref = to;
  }
};

__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));       // a NaN is passed over
  return y;
}

// All threads receive the statistics of the CTA, or of the cluster's CTAs that share a row.  The maximum goes first, so that every
// thread rescales its sums once.  `scratch`: 100 floats.  A cluster's CTAs must not leave before all have come back from here (their
// shared memory is read): see cluster_done.
template <int THREADS, bool ENTROPY>
__device__ __forceinline__ void vocab_reduce(VocabStats& st, float scale, float* scratch, int parts) {
  constexpr int WARPS = THREADS / 32;
  static_assert(WARPS == 4 || (WARPS >= 8 && WARPS <= 16), "the second sum is over 4, 8 or 16 lanes");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = warp_max(st.m);
  if (lane == 0) scratch[warp] = m;
  __syncthreads();
  m = warp_max(lane < WARPS ? scratch[lane] : -INFINITY);
  st.refer(m, scale);
  float s = warp_reduce(st.s, SumOp()), a = ENTROPY ? warp_reduce(st.a, SumOp()) : 0.f;
  if (lane == 0) { scratch[32 + warp] = s; scratch[64 + warp] = a; }
  __syncthreads();
  s = lane < WARPS ? scratch[32 + lane] : 0.f;
  a = lane < WARPS ? scratch[64 + lane] : 0.f;
#pragma unroll
  for (int o = WARPS > 8 ? 8 : WARPS / 2; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    if constexpr (ENTROPY) a += __shfl_xor_sync(0xffffffffu, a, o);
  }
  st = {m, m, __shfl_sync(0xffffffffu, s, 0), __shfl_sync(0xffffffffu, a, 0)};
  if (parts > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    if (threadIdx.x == 0) { scratch[96] = st.m; scratch[97] = st.s; scratch[98] = st.a; }
    cluster.sync();
    const float* peer = cluster.map_shared_rank(scratch, lane < parts ? lane : 0);
    st = lane < parts ? VocabStats{peer[96], peer[96], peer[97], peer[98]} : VocabStats{-INFINITY, -INFINITY, 0.f, 0.f};
    st.m = warp_max(st.m);
    st.refer(st.m, scale);
    st.s = warp_reduce(st.s, SumOp());
    if constexpr (ENTROPY) st.a = warp_reduce(st.a, SumOp());
  }
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
  // Which thread of this part's CTA works on element `index`, -1: none.
  template <int THREADS, typename R> __device__ __forceinline__ int owner(const R& r, int index) const {
    const int e = index - r.head;
    if (e < 0) return part == 0 ? index : -1;
    const int v = e / R::kVec;
    if (v >= r.whole) return part == 0 ? r.head + index - (r.M - r.tail) : -1;
    return v >= lo && v < hi ? (v - lo) % THREADS : -1;
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

// Element j of a packet, j known at run time only.
template <typename T> __device__ __forceinline__ float packet_element(const Pack<T>& p, int j) {
  constexpr int LG = sizeof(T) == 2 ? 1 : 0;
  const uint32_t w = (j >> LG & 2) ? ((j >> LG & 1) ? p.raw.w : p.raw.z) : ((j >> LG & 1) ? p.raw.y : p.raw.x);
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(w);
  } else {
    const unsigned short h = (unsigned short)(w >> ((j & 1) * 16));
    return Elem<T>::to_f(*reinterpret_cast<const T*>(&h));
  }
}

// -Inf in every element.
template <typename T> __device__ __forceinline__ uint4 no_logits() {
  const uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  return make_uint4(w, w, w, w);
}

// One thread's running sums, in two chains (packed fp32 pairs).
template <typename T, bool ENTROPY> struct VocabSum {
  static constexpr int kVec = Elem<T>::kVec;
  float m = -INFINITY, ref = -INFINITY;
  float2 s = {0.f, 0.f}, a = {0.f, 0.f};

  __device__ __forceinline__ void first(float f, float scale) {       // a single element (a NaN or +Inf gives a NaN sum here as below)
    m = ref = fmaxf(m, f);
    s.x = vocab_ex2((f - (ref == -INFINITY ? 0.f : ref)) * scale);
  }
  template <int U> __device__ __forceinline__ float take(const Pack<T> (&p)[U], float scale) {       // returns the largest of the step
    const float most = packets_max<T, U>(p);
    m = fmaxf(m, most);
    if ((m - ref) * scale > kRefSlack) {              // (both -Inf: a NaN, no)
      const float d = fmaxf((ref - m) * scale, kExpFloor), e = vocab_ex2(d);
      if constexpr (ENTROPY) a = __fmul2_rn(make_float2(e, e), __ffma2_rn(make_float2(d, d), s, a));
      s = __fmul2_rn(make_float2(e, e), s);
      ref = m;
    }
    const float mo = ref == -INFINITY ? 0.f : -ref;
    const float2 nm = make_float2(mo, mo), sc = make_float2(scale, scale);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[kVec];
      p[u].unpack(f);
#pragma unroll
      for (int j = 0; j < kVec; j += 2) {
        const float2 y = __fmul2_rn(__fadd2_rn(make_float2(f[j], f[j + 1]), nm), sc);
        const float2 e = make_float2(vocab_ex2(y.x), vocab_ex2(y.y));
        s = __fadd2_rn(s, e);
        if constexpr (ENTROPY) a = __ffma2_rn(e, make_float2(fmaxf(y.x, kExpFloor), fmaxf(y.y, kExpFloor)), a);
      }
    }
    return most;
  }
  __device__ __forceinline__ VocabStats stats() const { return {m, ref, s.x + s.y, a.x + a.y}; }
};

// A CTA that is done with its row asks L2 for the first 32 KB of one that will be begun soon, so that memory has work while rows end
// and begin: three quarters of the CTAs that are under way at once further on.  2048 x 131072 bf16 86 us without, 78.7 so; with all of
// them further on 79.5, with 96 KB 79.5, with the whole row 94; 4096 x 32768 49.7 without, 44.0 so.  (Chunks of the CTA's own row ahead
// of its loads: 91.)  Under the power cap of longer runs nothing is left of it for 16-bit types; 777 x 50001 fp32, forward and
// backward, 84.5 and 83.3 us there.  Only where a CTA has a row to itself: few rows are under way all at once.
template <typename T> __device__ __forceinline__ void vocab_ask_ahead(const T* X, int64_t ldx, int M, size_t row, int ctas, int parts) {
  row += ctas - ctas / 4;
  if (parts > 1 || threadIdx.x || row >= gridDim.x) return;
  const T* x = X + row * ldx;
  const VocabRow<T> r(x, M);
  const uint32_t bytes = min(r.whole, 2048) * 16;
  if (bytes) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(x + r.head), "r"(bytes) : "memory");
}

// The largest logit of every cell of a thread's share: a cell is 2^shift consecutive steps, so that no share has more than kCells.
constexpr int kCells = 16;
template <int THREADS> struct VocabCells {
  float (*max)[THREADS];       // shared memory: kCells rows
  int shift, cells;
  __device__ __forceinline__ VocabCells(float (*max_)[THREADS], int packets, int per_step) : max(max_), shift(0) {
    const int steps = (packets + per_step - 1) / per_step;
    while ((steps - 1) >> shift >= kCells) ++shift;
    cells = steps > 0 ? ((steps - 1) >> shift) + 1 : 0;
  }
};

// One thread's share of a part: every THREADS-th packet, U at a time, and a single element.  KEEP: the part will be read again.
// CELLS: the largest logits of the cells are left in `cells` (the single element belongs to none).
template <typename T, int THREADS, int U, bool ENTROPY, bool KEEP, bool CELLS>
__device__ __forceinline__ VocabStats vocab_thread_stats(const T* x, const VocabRow<T>& r, const VocabPart& part, float scale,
                                                         const VocabCells<THREADS>* cells) {
  constexpr int VEC = Elem<T>::kVec;
  VocabSum<T, ENTROPY> sum;
  const int one = part.part == 0 ? r.single(threadIdx.x) : -1;
  if (one >= 0) sum.first(Elem<T>::to_f(x[one]), scale);
  const uint64_t keep = KEEP ? keep_policy() : 0;
  const T* q = x + r.index(part.lo + threadIdx.x);
  auto load = [&](Pack<T>& p, int u) {
    if constexpr (KEEP) p.raw = ld_logits(q + u * (THREADS * VEC), keep);
    else p.raw = ld_logits(q + u * (THREADS * VEC));
  };
  int left = part.hi - part.lo - (int)threadIdx.x;    // packets from this thread's next one to the part's end
  Pack<T> p[U];
  if constexpr (CELLS) {
    float most = -INFINITY;
    for (int c = 0, i = 0; c < cells->cells; ++i, left -= U * THREADS, q += U * THREADS * VEC) {
      if (left > (U - 1) * THREADS) {
#pragma unroll
        for (int u = 0; u < U; ++u) load(p[u], u);
        most = fmaxf(most, sum.take(p, scale));
      } else if (left > 0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (left > u * THREADS) load(p[u], u);
          else p[u].raw = no_logits<T>();
        }
        most = fmaxf(most, sum.take(p, scale));
      }
      if (((i + 1) & ((1 << cells->shift) - 1)) == 0 || (int)(left + threadIdx.x) <= U * THREADS) {     // the cell's, or the part's, last step
        cells->max[c++][threadIdx.x] = most;
        most = -INFINITY;
      }
    }
    return sum.stats();
  }
  for (; left > (U - 1) * THREADS; left -= U * THREADS, q += U * THREADS * VEC) {
#pragma unroll
    for (int u = 0; u < U; ++u) load(p[u], u);
    sum.take(p, scale);
  }
  if (left > 0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (left > u * THREADS) load(p[u], u);
      else p[u].raw = no_logits<T>();
    }
    sum.take(p, scale);
  }
  return sum.stats();
}

// The same for a part of at most THREADS * U * GROUPS packets that waits in shared memory for its second look.  Every thread asks for
// all of its packets at once, by asynchronous copies in GROUPS groups, and reads back nothing but its own: no barrier, no registers
// held by what is on its way.
__device__ __forceinline__ void wait_copies(int later) {       // until at most `later` groups of this thread's copies are on their way
  switch (later) {
#define TYLO_WAIT_COPIES(N) case N: asm volatile("cp.async.wait_group " #N ";" ::: "memory"); break;
    TYLO_WAIT_COPIES(0) TYLO_WAIT_COPIES(1) TYLO_WAIT_COPIES(2) TYLO_WAIT_COPIES(3)
    TYLO_WAIT_COPIES(4) TYLO_WAIT_COPIES(5) TYLO_WAIT_COPIES(6) TYLO_WAIT_COPIES(7)
#undef TYLO_WAIT_COPIES
  }
}
template <typename T, int THREADS, int U, int GROUPS>
__device__ __forceinline__ void vocab_resident_ask(uint4* row, const T* x, const VocabRow<T>& r, const VocabPart& part) {
  static_assert(GROUPS <= 8, "wait_copies");
  const int n = part.hi - part.lo - (int)threadIdx.x;          // this thread's packet k * THREADS is there if n > k * THREADS
  const T* q = x + r.index(part.lo + threadIdx.x);
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(row + threadIdx.x);
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (g * U + u) * THREADS;
      if (n > k) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + k * 16), "l"(q + k * Elem<T>::kVec) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
}
template <typename T, int THREADS, int U, int GROUPS, bool ENTROPY>
__device__ __forceinline__ VocabStats vocab_resident_stats(const uint4* row, const T* x, const VocabRow<T>& r, const VocabPart& part, float scale) {
  const int n = part.hi - part.lo - (int)threadIdx.x;
  const uint4* own = row + threadIdx.x;
  VocabSum<T, ENTROPY> sum;
  const int one = part.part == 0 ? r.single(threadIdx.x) : -1;
  if (one >= 0) sum.first(Elem<T>::to_f(x[one]), scale);
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    wait_copies(GROUPS - 1 - g);
    if (n > g * U * THREADS) {
      Pack<T> p[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = (g * U + u) * THREADS;
        p[u].raw = n > k ? own[k] : no_logits<T>();
      }
      sum.take(p, scale);
    }
  }
  return sum.stats();
}

// Special-function units: a fourth of the exponentials as polynomials on the multiply-add pipes was slower everywhere (bf16, ex2 alone and
// so: entropy of 4096 x 131072 169 and 181 us, value and gradient of 4096 x 32768 91 and 93), and one fused multiply-add per exponent
// against a rounded reference changed nothing: what is left is memory and, in longer runs, the power cap (1000 W, 1.76 GHz).

// Gradient of a part that waits in shared memory (vocab_resident_stats): f(pair of logits) -> pair of gradients for every element,
// rounded once, on the way out.
template <typename T, int THREADS, int U, typename F>
__device__ __forceinline__ void vocab_resident_rewrite(T* dx, const uint4* kept, const T* x, const VocabRow<T>& r, const VocabPart& part, F f) {
  constexpr int VEC = Elem<T>::kVec;
  const int one = part.part == 0 ? r.single(threadIdx.x) : -1;
  if (one >= 0) dx[one] = Elem<T>::from_f(f(make_float2(Elem<T>::to_f(x[one]), 0.f)).x);
  const int n = part.hi - part.lo;
  T* to = dx + r.index(part.lo);
#pragma unroll U
  for (int v = threadIdx.x; v < n; v += THREADS) {
    Pack<T> p;
    p.raw = kept[v];
    float e[VEC];
    p.unpack(e);
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      const float2 d = f(make_float2(e[j], e[j + 1]));
      e[j] = d.x; e[j + 1] = d.y;
    }
    p.pack(e);
    st_stream(to + (size_t)v * VEC, p.raw);
  }
}

// The same from global memory.  As the second look at a part it goes backwards: what was read last is the likeliest to be in L2.
template <typename T, int THREADS, int U, typename F>
__device__ __forceinline__ void vocab_rewrite(T* dx, const T* x, const VocabRow<T>& r, const VocabPart& part, F f) {
  constexpr int VEC = Elem<T>::kVec;
  const int one = part.part == 0 ? r.single(threadIdx.x) : -1;
  if (one >= 0) dx[one] = Elem<T>::from_f(f(make_float2(Elem<T>::to_f(x[one]), 0.f)).x);
  auto give = [&](Pack<T>& p, T* to) {
    float e[VEC];
    p.unpack(e);
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      const float2 d = f(make_float2(e[j], e[j + 1]));
      e[j] = d.x; e[j + 1] = d.y;
    }
    p.pack(e);
    st_stream(to, p.raw);
  };
  const uint64_t drop = drop_policy();
  const int n = part.hi - part.lo, steps = n / (U * THREADS);
  const int first = r.index(part.lo + threadIdx.x);
  {
    const int i = first + steps * (U * THREADS * VEC), left = n - steps * (U * THREADS) - (int)threadIdx.x;
    Pack<T> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (left > u * THREADS) p[u].raw = ld_logits(x + i + u * (THREADS * VEC), drop);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (left > u * THREADS) give(p[u], dx + i + u * (THREADS * VEC));
  }
  for (int k = steps - 1; k >= 0; --k) {
    const T* q = x + first + k * (U * THREADS * VEC);
    T* to = dx + first + k * (U * THREADS * VEC);
    Pack<T> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) p[u].raw = ld_logits(q + u * (THREADS * VEC), drop);
#pragma unroll
    for (int u = 0; u < U; ++u) give(p[u], to + u * (THREADS * VEC));
  }
}

// A gradient of zeros.
template <typename T, int THREADS>
__device__ __forceinline__ void vocab_zero(T* dx, const VocabRow<T>& r, const VocabPart& part) {
  const int one = part.part == 0 ? r.single(threadIdx.x) : -1;
  if (one >= 0) dx[one] = Elem<T>::from_f(0.f);
  for (int v = part.lo + threadIdx.x; v < part.hi; v += THREADS) st_stream(dx + r.index(v), make_uint4(0, 0, 0, 0));
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

// ---- the largest elements of a part ------------------------------------------------------------------------------------------
// A bound first: the K-th largest of the threads' own maxima, which the statistics leave behind, is no larger than the K-th largest
// element, and little more than K cells of all threads reach it.  Only those are read again, out of L2, and what reaches the bound goes
// to shared memory: little more than K elements unless many sit together in few shares or are equal.  Where they do not fit, the bound
// is raised by counting, and equal elements at the bound are taken in the order of their index.  What is left is thinned by bisection
// to K and a few, whose rank is counted.
// It is made for rows whose threads hold many more packets than K: where K is a large part of the elements the bound discards little, and the
// thinning, some thirty steps with up to four barriers each, is most of the time (figures in logprob.cu).
constexpr int kRanked = TYLO_TOP_MAX + 32;       // most elements that are ranked: lists of 32, one more than can be asked for

template <int THREADS> struct TopScratch {
  static constexpr int kSlots = 4 * THREADS;
  uint64_t keys[kSlots], few[kRanked];
  uint64_t sorted[TYLO_TOP_MAX];
  float cells[kCells][THREADS];
  uint32_t mine[THREADS];                 // the threads' largest elements as keys
  uint32_t warp[64], bound, most, dense;
  uint16_t hits[THREADS / 32][64];
  int rank[TYLO_TOP_MAX];
  int n, m;
};

template <int THREADS> struct BlockCount {
  // sum over the CTA; `buf` alternates between two halves so that one barrier per sum is enough
  uint32_t* buf;
  int half;
  __device__ __forceinline__ int operator()(int c) {
    c = __reduce_add_sync(0xffffffffu, c);
    uint32_t* b = buf + 32 * half;
    half ^= 1;
    if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = c;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    return __reduce_add_sync(0xffffffffu, lane < THREADS / 32 ? (int)b[lane] : 0);
  }
};

// Puts the min(K, elements of the part) largest elements of the part into sc.sorted, in falling order, and returns how many.
// sc.mine[thread]: the thread's largest element as a key, 0 without elements, written before a barrier of the CTA; `cells`: see
// vocab_thread_stats<U>; `all`: this thread's cells cannot be relied on (a NaN, which their maxima pass over).
template <typename T, int THREADS, int U>
__device__ __noinline__ int vocab_top(const T* x, const VocabRow<T> r, const VocabPart part, int K, VocabCells<THREADS> cells, bool all,
                                      TopScratch<THREADS>& sc) {
  constexpr int VEC = Elem<T>::kVec, kTopSlots = TopScratch<THREADS>::kSlots;
  uint64_t *keys = sc.keys, *few = sc.few;
  const int elements = (part.hi - part.lo) * VEC + (part.part == 0 ? r.head + r.tail : 0);
  K = min(K, elements);
  BlockCount<THREADS> count{sc.warp, 0};
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t mine = sc.mine[threadIdx.x];
  if (warp == 0) {
    // one warp looks for the bound, by bisection between the smallest and the largest maximum; a few more than K will do
    uint32_t k[THREADS / 32], hi = 0, lo = 0xffffffffu;
    int live = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
      k[i] = sc.mine[i * 32 + lane];
      hi = max(hi, k[i]);
      lo = min(lo, k[i] - 1);               // (0 becomes the largest)
      live += k[i] != 0;
    }
    hi = __reduce_max_sync(0xffffffffu, hi);
    lo = __reduce_min_sync(0xffffffffu, lo) + 1;
    const uint32_t most = hi;
    int reach = __reduce_add_sync(0xffffffffu, live);
    if (reach >= K) {
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        int c = 0;
#pragma unroll
        for (int i = 0; i < THREADS / 32; ++i) c += k[i] >= mid;
        c = __reduce_add_sync(0xffffffffu, c);
        if (c >= K) {
          lo = mid;
          reach = c;
          if (c <= K + K / 32 + 2) break;
        } else {
          hi = mid - 1;
        }
      }
    } else {
      // fewer threads hold data than K: the key of the smallest value.  The bound, and every bound raised from it, has to be a number's
      // key or lie above all numbers': a NaN's below it would compare as false with every cell.
      lo = vocab_key(-INFINITY);
    }
    // Many maxima equal to the bound, as where a mask leaves little: its equals would not fit, so they are not tried.  That many threads
    // must hold data: it can be seen so for K up to 48, 112 and 240 with 128, 256 and 512 of them; for more the equals are collected until
    // the places are full, and counted off then.
    if (lane == 0) { sc.bound = lo; sc.most = most; sc.dense = reach >= 2 * K + 32; sc.n = 0; sc.m = 0; }
  }
  __syncthreads();
  uint32_t t = sc.bound, lo, hi;
  const uint32_t top = sc.most;
  // Hands the elements of the cells whose maximum reaches `from` to f(packet, its elements as bits, index of the first) by the packet: a
  // warp lists such cells of its threads and deals their packets over its lanes.  f returns false when it has seen enough.
  auto visit = [&](uint32_t from, auto f) {
    bool more = true;
    const int one = part.part == 0 ? r.single(threadIdx.x) : -1;
    if (one >= 0) {
      Pack<T> p;
      float e[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) e[j] = Elem<T>::to_f(x[one]);
      p.pack(e);
      more = f(p, 1u, one);
    }
    const bool any = mine >= from;
    if (!__any_sync(0xffffffffu, any)) return;
    const float low = vocab_unkey(from);       // (above the key of +Inf it is a NaN: `all` alone counts)
    uint16_t* hits = sc.hits[warp];
    static_assert(U == 4, "packets of a cell as a power of two");
    const int lg = cells.shift + 2, per = 1 << lg;
    for (int c = 0; c < cells.cells;) {
      int n = 0;
      for (; c < cells.cells && n <= 32; ++c) {
        const bool hit = any && (all || cells.max[c][threadIdx.x] >= low);
        const uint32_t mask = __ballot_sync(0xffffffffu, hit);
        if (hit) hits[n + __popc(mask & ((1u << lane) - 1))] = (uint16_t)(c * 32 + lane);
        n += __popc(mask);
      }
      __syncwarp();
      for (int i0 = lane; i0 < n * per && more; i0 += 4 * 32) {
        Pack<T> p[4];
        int v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = i0 + u * 32, h = i < n * per ? hits[i >> lg] : 0;
          v[u] = part.lo + ((h >> 5) * per + (i & (per - 1))) * THREADS + warp * 32 + (h & 31);
          if (i >= n * per) v[u] = part.hi;
          if (v[u] < part.hi) p[u].raw = ld_logits(x + r.index(v[u]));
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (v[u] < part.hi && more) more = f(p[u], (1u << VEC) - 1, r.index(v[u]));
      }
      __syncwarp();
    }
  };
  // elements above or at a bound into sc.keys; more than kTopSlots: at least that many
  auto collect = [&](uint32_t from) {
    const float low = vocab_unkey(from);
    visit(from, [&](const Pack<T>& p, uint32_t there, int first) {
      float e[VEC];
      p.unpack(e);
      uint32_t hit = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) hit |= (uint32_t)!(e[j] < low) << j;
      for (hit &= there; hit; hit &= hit - 1) {
        const int j = __ffs(hit) - 1;
        const uint64_t k = vocab_key(packet_element(p, j), first + j);
        if ((uint32_t)(k >> 32) < from) continue;             // NaN, and bounds without a value of their own
        const int at = atomicAdd(&sc.n, 1);
        if (at >= kTopSlots) return false;
        keys[at] = k;
      }
      return true;
    });
    __syncthreads();
    return sc.n;
  };
  auto at_least = [&](uint32_t from) {
    int c = 0;
    visit(from, [&](const Pack<T>& p, uint32_t there, int) {
      for (uint32_t b = there; b; b &= b - 1) c += vocab_key(packet_element(p, __ffs(b) - 1)) >= from;
      return true;
    });
    return count(c);
  };
  auto clear = [&]() {
    __syncthreads();
    if (threadIdx.x == 0) sc.n = 0;
    __syncthreads();
  };
  auto above = [&](uint32_t bound) { return bound == 0xffffffffu ? 0 : collect(bound + 1); };     // nothing is above a NaN
  int n = sc.dense ? kTopSlots + 1 : collect(t);
  if (n > kTopSlots) {
    clear();
    n = above(t);
    if (n > kTopSlots) {                       // raise it: at_least(lo) >= K, at_least(hi + 1) < K
      lo = t + 1; hi = top;
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        const int c = at_least(mid);
        if (c >= K) {
          lo = mid;
          if (c <= kTopSlots) break;
        } else {
          hi = mid - 1;
        }
      }
      t = lo;
      clear();
      n = collect(t);
      if (n > kTopSlots) { clear(); n = above(t); }
    }
    if (n < K) {       // (at least K elements reach t, whichever way it was found)
      // the elements equal to the bound, lowest index first: they are counted off in blocks of THREADS packets
      const int need = K - n;
      int taken = 0;
      auto block = [&](uint32_t ties, int first) {        // bit j: element first + j
        const int c = __popc(ties);
        int before = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += up;
        }
        if (lane == 31) sc.warp[threadIdx.x >> 5] = before;
        __syncthreads();
        int ahead = 0, all = 0;
        for (int w = 0; w < THREADS / 32; ++w) {
          const int k = sc.warp[w];
          ahead += w < (int)(threadIdx.x >> 5) ? k : 0;
          all += k;
        }
        __syncthreads();
        int rank = taken + ahead + before - c;
        for (uint32_t b = ties; b && rank < need; b &= b - 1, ++rank)
          keys[n + rank] = ((uint64_t)t << 32) | (uint32_t)(0x7fffffff - (first + __ffs(b) - 1));
        taken += all;
      };
      if (part.part == 0 && r.head) block((int)threadIdx.x < r.head && vocab_key(Elem<T>::to_f(x[threadIdx.x])) == t, threadIdx.x);
      for (int v0 = part.lo; v0 < part.hi && taken < need; v0 += THREADS) {
        const int v = v0 + threadIdx.x;
        uint32_t ties = 0;
        if (v < part.hi) {
          Pack<T> p;
          p.raw = ld_logits(x + r.index(v));
          float e[VEC];
          p.unpack(e);
#pragma unroll
          for (int j = 0; j < VEC; ++j) ties |= (uint32_t)(vocab_key(e[j]) == t) << j;
        }
        block(ties, r.index(v));
      }
      if (part.part == 0 && r.tail && taken < need)
        block((int)threadIdx.x < r.tail && vocab_key(Elem<T>::to_f(x[r.M - r.tail + threadIdx.x])) == t, r.M - r.tail + threadIdx.x);
      n = K;
      __syncthreads();
    }
  }
  // n >= K different keys: thin them if they are many, then rank them
  uint64_t* list = keys;
  if (n > kRanked) {
    constexpr int PER = kTopSlots / THREADS;
    uint64_t mine64[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) mine64[i] = i * THREADS + threadIdx.x < n ? keys[i * THREADS + threadIdx.x] : 0;
    uint64_t lo64 = (uint64_t)t << 32, hi64 = ((uint64_t)top << 32) | 0xffffffffu;
    while (lo64 < hi64) {
      const uint64_t mid = lo64 + (hi64 - lo64) / 2 + 1;
      int c = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i * THREADS < n) c += __syncthreads_count(mine64[i] >= mid);
      if (c >= K) {
        lo64 = mid;
        if (c <= kRanked) break;
      } else {
        hi64 = mid - 1;
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (mine64[i] >= lo64) few[atomicAdd(&sc.m, 1)] = mine64[i];
    __syncthreads();
    n = sc.m;
    list = few;
  }
  // every warp sorts 32 of them; a key's rank is its place there and the number of larger keys in each of the other sorted lists
  const int lists = (n + 31) / 32;
  for (int l = warp; l < lists; l += THREADS / 32) {
    uint64_t k = l * 32 + lane < n ? list[l * 32 + lane] : 0;
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
      for (int step = size / 2; step > 0; step /= 2) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, k, step);
        const bool larger = ((lane & step) == 0) == ((lane & size) == 0 || size == 32);      // falling order in the end
        if ((other > k) == larger) k = other;
      }
    list[l * 32 + lane] = k;
  }
  __syncthreads();
  for (int l = warp; l < lists; l += THREADS / 32) {
    const uint64_t k = list[l * 32 + lane];
    int rank = lane;
    for (int o = 0; o < lists; ++o) {
      if (o == l) continue;
      const uint64_t* other = list + o * 32;
      int larger = 0;
#pragma unroll
      for (int step = 16; step > 0; step /= 2)
        if (other[larger + step - 1] > k) larger += step;
      rank += larger + (other[larger] > k);
    }
    if (k && rank < K) sc.sorted[rank] = k;
  }
  __syncthreads();
  return K;
}

// Hands every one of the row's `K` largest elements to f(rank, key), whichever CTA of the row's cluster holds it (n of them in
// sc.sorted here): its rank is its place in its own list and, for every other list, the number of larger elements there (lists are
// sorted: a binary search, a thread for each element and list).  The lists are fetched once: a search in another CTA's memory would
// wait for it at every step (one row of 32768, 20 alternatives: 16.2 us).
template <int THREADS, typename F>
__device__ __forceinline__ void vocab_ranked(TopScratch<THREADS>& sc, int n, int K, int parts, F f) {
  if (parts == 1) {
    for (int i = threadIdx.x; i < n; i += THREADS) f(i, sc.sorted[i]);
    return;
  }
  cg::cluster_group cluster = cg::this_cluster();
  const int me = cluster.block_rank();
  for (int i = n + threadIdx.x; i < K; i += THREADS) sc.sorted[i] = 0;
  cluster.sync();
  uint64_t* all = sc.keys;                       // parts * K of its 4 * THREADS places (the launch sees to it)
  for (int i = threadIdx.x; i < parts * K; i += THREADS) all[i] = cluster.map_shared_rank(&sc, i / K)->sorted[i % K];
  for (int i = threadIdx.x; i < K; i += THREADS) sc.rank[i] = i;
  __syncthreads();
  for (int i = threadIdx.x; i < parts * K; i += THREADS) {
    const int c = i / K, j = i % K;
    if (c == me || j >= n) continue;
    const uint64_t k = sc.sorted[j];
    int lo = 0, hi = K;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (all[c * K + mid] > k) lo = mid + 1; else hi = mid;
    }
    atomicAdd(&sc.rank[j], lo);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += THREADS)
    if (sc.rank[i] < K) f(sc.rank[i], sc.sorted[i]);
}

// This thread's largest element as a key; a NaN counts, so a share whose sum is NaN is looked through.
template <typename T, int THREADS>
__device__ __forceinline__ uint32_t vocab_mine(const T* x, const VocabRow<T>& r, const VocabPart& part, const VocabStats& st) {
  uint32_t k = 0;
  const int one = part.part == 0 ? r.single(threadIdx.x) : -1;
  if (st.s != st.s) {
    if (one >= 0) k = vocab_key(Elem<T>::to_f(x[one]));
    for (int v = part.lo + threadIdx.x; v < part.hi; v += THREADS)
      for (int j = 0; j < Elem<T>::kVec; ++j) k = max(k, vocab_key(Elem<T>::to_f(x[r.index(v) + j])));
  } else if (part.lo + (int)threadIdx.x < part.hi || one >= 0) {
    k = vocab_key(st.m);
  }
  return k;
}

// Rows of up to this many packets per CTA wait in shared memory for their second look: 106 KB, two CTAs per SM (one, where more than
// about 560 entries of a teacher lie before a row of that length).
constexpr int kResident = 6784;
// Most dynamic shared memory of a launch: such a row with its teacher's entries.  Where a kernel may need more than the default, the limit
// is raised to this, not to what the call needs: calls of other sizes may be under way on other threads between the raise and the launch.
constexpr int kVocabMaxShared = kResident * 16 + 12 * TYLO_DISTILL_MAX;
static_assert(sizeof(TopScratch<512>) <= kVocabMaxShared, "alternatives");

// Launches `parts` CTAs per row, as a cluster where they have something to tell one another.
template <typename A>
int32_t launch_vocab(const char* who, void (*kernel)(A, int), const A& args, int64_t N, int parts, int threads, cudaStream_t stream, int smem = 0) {
  if (smem > 40 * 1024)       // (with the kernels' own arrays; the default limit is 48 KB)
    TYLO_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kVocabMaxShared));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(N * parts));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args, parts);
  if (e != cudaSuccess) {
    cudaGetLastError();                     // it is told here: the next launch's check is not to find it
    set_error("launch of %s failed: %s", who, cudaGetErrorString(e));
    return TYLO_ERR_CUDA;
  }
  return TYLO_OK;
}

// CTAs per row: a row is dealt over a cluster while rows alone leave SMs without a CTA.  Forward, bf16, us with 1 / 2 / 4 CTAs per row: 148 x
// 131072 14.2 / 15.5 / 15.2, with 20 alternatives 27.0 / 23.2 / 22.2; 300 x 131072 21.8 / 21.3 / 19.7, with 20 alternatives 29.3 / 27.9 /
// 33.6; 600 x 65536 21.4 / 23.8 / 25.7; 512 x 262144 49.7 / 51.7 / 52.1.
inline int vocab_parts(int64_t N, int64_t packets) {
  int parts = 1;
  while (parts < 8 && N * parts * 2 <= 2 * sm_count() && packets >= parts * 1024LL) parts *= 2;
  return parts;
}
// The same for kernels that look at their row twice: rows longer than `pair` packets go to two CTAs, so that fewer of them are under way
// and the second look finds more in L2.  Value and gradient, bf16, us with one CTA / two: log probabilities 2048 x 100,000 157 / 165,
// 2048 x 131,072 213 / 193, 2048 x 262,144 458 / 420; distillation 4096 x 131,072 425 / 433, 2048 x 200,000 359 / 329.
inline int vocab_parts_twice(int64_t N, int64_t packets, int64_t pair) {
  const int parts = vocab_parts(N, packets);
  return packets > pair && parts < 2 ? 2 : parts;
}

// Shape of a kernel that looks at its row once, by the packets of a CTA.
#define TYLO_VOCAB_STREAM(LAUNCH)        \
  if (per <= 2048) return LAUNCH(128);   \
  if (per <= 8192) return LAUNCH(256);   \
  return LAUNCH(512)

// Shape of a kernel that looks at its row twice: rows of up to kResident packets per CTA wait in shared memory.  Value and gradient, bf16, us,
// waiting / read again: 8192 x 16000 81 / 90, 4096 x 32768 83 / 93, 2048 x 50000 75 / 77.
#define TYLO_VOCAB_RESIDENT(LAUNCH)                                      \
  if (per <= 1024) return LAUNCH(128, 4, 2);                             \
  if (per <= 2048) return LAUNCH(128, 4, 4);                             \
  if (per <= 4096) return LAUNCH(256, 4, 4);                             \
  if (per <= kResident) return LAUNCH(512, 2, 7);                        \
  return LAUNCH(512, 4, 0)

// The gradient of N rows of M logits, rows ldx apart, is written over the logits themselves or anywhere beside them.
inline int32_t check_vocab_grad(const char* who, const void* dX, const void* X, int64_t M, int64_t N, int64_t ldx, int32_t dtype) {
  TYLO_REQUIRE(dX, TYLO_ERR_INVALID_ARGUMENT, "%s: dX must be non-null", who);
  TYLO_REQUIRE(aligned16(dX), TYLO_ERR_MISALIGNED, "%s: dX must be 16-byte aligned", who);
  const int64_t apart = ((const char*)dX - (const char*)X) / (dtype == TYLO_F32 ? 4 : 2), within = (apart % ldx + ldx) % ldx;
  const bool far = apart >= (N - 1) * ldx + M || -apart >= (N - 1) * ldx + M;
  TYLO_REQUIRE(apart == 0 || far || (within >= M && ldx - within >= M), TYLO_ERR_INVALID_ARGUMENT,
               "%s: dX must be X or not overlap it", who);
  return TYLO_OK;
}

inline int32_t check_vocab(const char* who, const void* X, int64_t M, int64_t N, int64_t ldx, float temperature) {
  TYLO_REQUIRE(X, TYLO_ERR_INVALID_ARGUMENT, "%s: X must be non-null", who);
  TYLO_REQUIRE(M > 0 && N > 0, TYLO_ERR_INVALID_ARGUMENT, "%s: extents must be positive (M=%lld, N=%lld)", who, (long long)M,
               (long long)N);
  TYLO_REQUIRE(ldx >= M, TYLO_ERR_INVALID_ARGUMENT, "%s: ldx (%lld) must be at least M (%lld)", who, (long long)ldx, (long long)M);
  TYLO_REQUIRE(M < 0x7fff0000LL && N <= 0x0fffffffLL && ldx <= 1LL << 34, TYLO_ERR_UNSUPPORTED,
               "%s: M from 2^31-2^16, N above 2^28-1 or ldx above 2^34 is not supported", who);
  TYLO_REQUIRE(temperature > 0.f && temperature <= 3.0e38f && 1.f / temperature <= 1e30f, TYLO_ERR_INVALID_ARGUMENT,
               "%s: temperature must be positive and finite", who);
  TYLO_REQUIRE(aligned16(X), TYLO_ERR_MISALIGNED, "%s: X must be 16-byte aligned", who);
  return TYLO_OK;
}

}  // namespace tylo
