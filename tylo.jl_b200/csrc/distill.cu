// Distillation from a teacher's top logits, and its gradient.  With q = softmax(x / t) of the student's row and the teacher's K
// entries (value v_k at index I_k, temperature u), p_k = exp(v_k / u) / sum_j exp(v_j / u), or exp(v_k / u) as it is where the
// teacher's own mass is kept:
//
//   loss = sum_k p_k (log p_k - log q_{I_k})
//   dX_j = w / t (P q_j - sum_{k: I_k = j} p_k),   P = sum_k p_k
//
// Entries with an index outside [0, M) are left out, of the teacher's normalisation too.
//
// Bound, shapes and how times are taken as in logprob.cu; the entries come on top.  us, bf16: the loss with 64 entries 2048 x 131072 96, 4096 x
// 65536 96, 512 x 131072 29; of 4096 x 32768 with 1 52, with 128 58.  Value and gradient of 4096 x 32768 with 1 / 128 / 256 / 512 / 1,024
// entries 103 / 120 / 147 / 270 / 936, of 4096 x 131072 with 1 / 128 / 1,024 431 / 445 / 915: every entry is compared with every other for
// copies of its index.  The backward with 1 and 128 entries: 4096 x 32768 91 and 107, 4096 x 65536 171 and 195.  The entries
// of a row are dealt with by one warp, so their sums are the same for every shape; an index that occurs more than once is summed in
// the order of the entries by whoever stores it, so no order of the GPU's shows.
#include "vocab.cuh"

namespace tylo {

struct DistillArgs {
  const void* X;
  const float* teacher;
  const int32_t* index;
  float *Loss, *Mx, *L;
  void* dX;
  const float* dLoss;
  const float *inMx, *inL;
  int64_t ldx;
  int M, K, renormalize, sms;
  float temperature, teacher_temperature;
};

// Places for K entries in each of the three arrays, so that what follows them is 16-byte aligned.
__host__ __device__ constexpr int entry_slots(int K) { return (K + 3) / 4 * 4; }

// A row's entries in shared memory.
struct Entries {
  float *p, *xk;         // the teacher's value, then its probability; the student's logit
  int* index;            // -1: left out
  __device__ __forceinline__ Entries(void* space, int slots)
      : p(reinterpret_cast<float*>(space)), xk(p + slots), index(reinterpret_cast<int*>(xk + slots)) {}
};

// Entries `first`, `first + STEP`, ... of a row, four asked for at a time.  The logits are read before any gradient is written (dX may
// be X).
template <typename T, int STEP>
__device__ __forceinline__ void load_entries(const DistillArgs& a, const Entries& e, size_t row, const T* x, int first, int slots) {
  const float* teacher = a.teacher + row * a.K;
  const int32_t* ids = a.index + row * a.K;
  for (int k0 = first; k0 < slots; k0 += 4 * STEP) {
    int id[4];
    float value[4], logit[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = k0 + i * STEP;
      id[i] = k < a.K ? ids[k] : -1;
      value[i] = k < a.K ? teacher[k] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (id[i] >= a.M) id[i] = -1;
      logit[i] = id[i] >= 0 ? Elem<T>::to_f(x[id[i]]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = k0 + i * STEP;
      if (k >= slots) break;
      e.index[k] = id[i] >= 0 ? id[i] : -1;
      e.p[k] = id[i] >= 0 ? value[i] : -INFINITY;
      e.xk[k] = logit[i];
    }
  }
}

// By one warp, all lanes: probabilities exp((v_k - m) / u) / S from values v_k (the difference first: the lowest value overflows where it
// is divided by less than 1; a factor 1 / u, for a quotient of each entry costs 10 us of 50 for 4096 x 32768 bf16 with 128);
// returns their sum, and m and log S.
__device__ __forceinline__ float teacher_probabilities(const DistillArgs& a, const Entries& e, float& m, float& log_sum) {
  const int lane = threadIdx.x & 31;
  const float iu = 1.f / a.teacher_temperature;
  m = log_sum = 0.f;
  if (a.renormalize) {
    float most = -INFINITY;
    for (int k = lane; k < a.K; k += 32) most = fmaxf(most, e.p[k]);
    most = warp_max(most);
    m = most == -INFINITY ? 0.f : most;
  }
  float sum = 0.f;
  for (int k = lane; k < a.K; k += 32) {
    const float p = expf((e.p[k] - m) * iu);
    e.p[k] = p;
    sum += p;
  }
  sum = warp_reduce(sum, SumOp());
  if (!a.renormalize || sum == 0.f) return sum;
  log_sum = logf(sum);
  const float inv = 1.f / sum;
  for (int k = lane; k < a.K; k += 32) e.p[k] *= inv;
  return sum * inv;
}

// Threads beside those that work on the row: where value and gradient are computed together, a warp of its own has the entries ready
// by the time the sums are (on one of the row's warps, before or after its share of the sums, all others wait for it: 4096 x 32768 bf16
// with 128 entries 137 and 120 us).
constexpr int distill_extra(bool loss, bool grad) { return loss && grad ? 32 : 0; }
constexpr int distill_ctas(int threads, int groups, bool grad) {
  return groups ? (threads == 128 ? 7 : threads == 256 ? 4 : 2) : 512 / threads * (grad ? 3 : 4);     // (480: 1)
}

// GROUPS > 0: the part waits in shared memory for the second look.  Dynamic shared memory: the entries, then the part.
template <typename T, int THREADS, int U, int GROUPS, bool LOSS, bool GRAD>
__global__ void __launch_bounds__(THREADS + distill_extra(LOSS, GRAD), distill_ctas(THREADS, GROUPS, GRAD))
distill_row_kernel(const DistillArgs a, int parts) {
  constexpr bool EXTRA = distill_extra(LOSS, GRAD) > 0;
  __shared__ float scratch[100];
  extern __shared__ uint4 dynamic[];
  const int slots = entry_slots(a.K);
  const Entries e(dynamic, slots);
  uint4* kept = reinterpret_cast<uint4*>(e.index + slots);
  // (the gradient alone goes from the last row to the first: what the forward read last is still in L2)
  const unsigned block = LOSS ? blockIdx.x : gridDim.x - 1 - blockIdx.x;
  const size_t row = block / parts;
  const T* x = (const T*)a.X + row * a.ldx;
  const VocabRow<T> r(x, a.M);
  const VocabPart part(block % parts, parts, r.whole);
  const float scale = kVocabLog2e / a.temperature;
  const bool on_row = !EXTRA || threadIdx.x < THREADS;
  const bool on_entries = EXTRA ? threadIdx.x >= THREADS : threadIdx.x < 32;      // a warp
  const int lane = threadIdx.x & 31;
  float w = 0.f, teacher_max = 0.f, teacher_log = 0.f;
  if constexpr (GRAD) w = a.dLoss[row] / a.temperature;
  VocabStats st{-INFINITY, -INFINITY, 0.f, 0.f};
  if (on_row) {
    if constexpr (GROUPS > 0) {
      vocab_resident_ask<T, THREADS, U, GROUPS>(kept, x, r, part);
      st = vocab_resident_stats<T, THREADS, U, GROUPS, false>(kept, x, r, part, scale);
    } else if constexpr (LOSS) {
      st = vocab_thread_stats<T, THREADS, U, false, GRAD, false>(x, r, part, scale, nullptr);
    } else {
      st = {a.inMx[row], 0.f, a.inL[row], 0.f};
    }
  }
  auto probabilities = [&]() {
    const float mass = teacher_probabilities(a, e, teacher_max, teacher_log);
    if (lane == 0) scratch[99] = mass;
  };
  if constexpr (EXTRA) {
    if (on_entries) {
      load_entries<T, 32>(a, e, row, x, lane, slots);
      __syncwarp();
      probabilities();
    }
    vocab_reduce<THREADS, false>(st, scale, scratch, parts);      // its barriers publish the entries
  } else {
    load_entries<T, THREADS>(a, e, row, x, threadIdx.x, slots);
    // (long rows only: 2048 x 131072 bf16 with 64 entries 87 us without and 83 so, but 4096 x 65536 87 and 94, 8192 x 16000 52 and 57)
    if constexpr (LOSS && THREADS == 512) vocab_ask_ahead((const T*)a.X, a.ldx, a.M, row, a.sms * distill_ctas(THREADS, GROUPS, GRAD), parts);
    if constexpr (LOSS) vocab_reduce<THREADS, false>(st, scale, scratch, parts);
    else __syncthreads();
    if (on_entries && (GRAD || part.part == 0)) probabilities();
    if constexpr (GRAD) __syncthreads();
  }
  const float mo = st.m == -INFINITY ? 0.f : st.m;
  if (LOSS && on_entries && part.part == 0) {
    const float logL = st.s == 0.f ? 0.f : logf(st.s);
    const float* teacher = a.teacher + row * a.K;
    const float it = 1.f / a.temperature, iu = 1.f / a.teacher_temperature;     // (here: no registers for them in the loops above)
    float loss = 0.f;
    for (int k = lane; k < a.K; k += 32) {
      const float p = e.p[k];
      if (e.index[k] >= 0 && p != 0.f) loss += p * (((teacher[k] - teacher_max) * iu - teacher_log) - ((e.xk[k] - mo) * it - logL));
    }
    loss = warp_reduce(loss, SumOp());
    if (lane == 0) {
      a.Loss[row] = loss;
      if (a.Mx) { a.Mx[row] = st.m; a.L[row] = st.s; }
    }
  }
  if constexpr (GRAD) {
    const float mass = scratch[99];
    T* dx = (T*)a.dX + row * a.ldx;
    if (w == 0.f || mass == 0.f || st.s == 0.f) {       // no weight, no teacher or no probability anywhere
      if (on_row) vocab_zero<T, THREADS>(dx, r, part);
    } else {
      const float2 m2 = make_float2(-mo, -mo), sc = make_float2(scale, scale), c = make_float2(w * mass / st.s, w * mass / st.s);
      auto grad = [&](float2 f) {
        const float2 y = __fmul2_rn(__fadd2_rn(f, m2), sc);
        return __fmul2_rn(make_float2(vocab_ex2(y.x), vocab_ex2(y.y)), c);
      };
      if (on_row) {
        if constexpr (GROUPS > 0) vocab_resident_rewrite<T, THREADS, U>(dx, kept, x, r, part, grad);
        else vocab_rewrite<T, THREADS, U>(dx, x, r, part, grad);
      }
      __syncthreads();
      // the teacher's entries in this part: every copy of an index sums all its copies in the same order and stores the same value
      const int4* four = reinterpret_cast<const int4*>(e.index);
      for (int k = threadIdx.x; k < a.K; k += THREADS + distill_extra(LOSS, GRAD)) {
        const int j = e.index[k];
        if (j < 0 || part.template owner<THREADS>(r, j) < 0) continue;
        float sum = 0.f;
        for (int i = 0; i < slots / 4; ++i) {
          const int4 q = four[i];
          if (q.x == j) sum += e.p[4 * i];
          if (q.y == j) sum += e.p[4 * i + 1];
          if (q.z == j) sum += e.p[4 * i + 2];
          if (q.w == j) sum += e.p[4 * i + 3];
        }
        dx[j] = Elem<T>::from_f(grad(make_float2(e.xk[k], 0.f)).x - w * sum);
      }
    }
  }
  if constexpr (LOSS) cluster_done(parts);
}

template <typename T, bool LOSS, bool GRAD>
static int32_t distill_dispatch(const char* who, const DistillArgs& a, int64_t N, cudaStream_t stream) {
  const int64_t packets = a.M / Elem<T>::kVec;
  const int entries = 12 * entry_slots(a.K);
  if constexpr (!LOSS) {
    // nothing to tell one another: plain CTAs of 4,096 packets, of 1,024 where the rows are few
    int64_t parts = (packets + 4095) / 4096;
    if (N * parts < 8 * sm_count()) parts = (packets + 1023) / 1024;
    parts = parts > 0 ? parts : 1;
    if (packets <= 1024) distill_row_kernel<T, 128, 4, 0, LOSS, GRAD><<<(unsigned)N, 128, entries, stream>>>(a, 1);
    else distill_row_kernel<T, 256, 4, 0, LOSS, GRAD><<<(unsigned)(N * parts), 256, entries, stream>>>(a, (int)parts);
    return check_launch(who);
  } else {
    const int parts = GRAD ? vocab_parts_twice(N, packets, 20480) : vocab_parts(N, packets);
    const int64_t per = (packets + parts - 1) / parts;
    if constexpr (!GRAD) {
#define TYLO_FWD(THREADS) launch_vocab(who, distill_row_kernel<T, THREADS, 4, 0, LOSS, GRAD>, a, N, parts, THREADS, stream, entries)
      TYLO_VOCAB_STREAM(TYLO_FWD);
#undef TYLO_FWD
    } else {
      // (without groups 480 threads: with the entries' warp 512, three times 40 registers)
#define TYLO_BOTH(THREADS, U, GROUPS)                                                                                                  \
  launch_vocab(who, distill_row_kernel<T, GROUPS ? THREADS : 480, U, GROUPS, LOSS, GRAD>, a, N, parts, (GROUPS ? THREADS : 480) + 32,  \
               stream, entries + (GROUPS ? (int)per * 16 : 0))
      TYLO_VOCAB_RESIDENT(TYLO_BOTH);
#undef TYLO_BOTH
    }
  }
}

}  // namespace tylo

using namespace tylo;

static int32_t check_distill(const char* who, const void* X, const float* teacher, const int32_t* index, int32_t K, int64_t M, int64_t N,
                             int64_t ldx, float temperature, float teacher_temperature) {
  if (int32_t rc = check_vocab(who, X, M, N, ldx, temperature)) return rc;
  TYLO_REQUIRE(teacher && index, TYLO_ERR_INVALID_ARGUMENT, "%s: teacher and index must be non-null", who);
  TYLO_REQUIRE(K > 0 && K <= TYLO_DISTILL_MAX, TYLO_ERR_INVALID_ARGUMENT, "%s: K (%d) must be between 1 and %d", who, K, TYLO_DISTILL_MAX);
  TYLO_REQUIRE(teacher_temperature > 0.f && teacher_temperature <= 3.0e38f && 1.f / teacher_temperature <= 1e30f,
               TYLO_ERR_INVALID_ARGUMENT, "%s: teacher_temperature must be positive and finite", who);
  return TYLO_OK;
}

static DistillArgs distill_args(const void* X, const float* teacher, const int32_t* index, int32_t K, int64_t M, int64_t ldx,
                                float temperature, float teacher_temperature, int32_t renormalize) {
  DistillArgs a = {};
  a.X = X; a.teacher = teacher; a.index = index; a.K = K; a.M = (int)M; a.ldx = ldx; a.sms = sm_count();
  a.temperature = temperature; a.teacher_temperature = teacher_temperature; a.renormalize = renormalize;
  return a;
}

extern "C" int32_t tylo_b200_distill_fwd(float* Loss, float* Mx, float* L, const void* X, const float* teacher, const int32_t* index,
                                         int32_t K, int64_t M, int64_t N, int64_t ldx, float temperature, float teacher_temperature,
                                         int32_t renormalize, int32_t dtype, tylo_stream_t stream) {
  const char* who = "distill_fwd";
  if (int32_t rc = check_distill(who, X, teacher, index, K, M, N, ldx, temperature, teacher_temperature)) return rc;
  TYLO_REQUIRE(Loss, TYLO_ERR_INVALID_ARGUMENT, "%s: Loss must be non-null", who);
  TYLO_REQUIRE(!Mx == !L, TYLO_ERR_INVALID_ARGUMENT, "%s: checkpoints Mx and L go together", who);
  DistillArgs a = distill_args(X, teacher, index, K, M, ldx, temperature, teacher_temperature, renormalize);
  a.Loss = Loss; a.Mx = Mx; a.L = L;
  TYLO_DISPATCH_DTYPE(dtype, T, return (distill_dispatch<T, true, false>(who, a, N, (cudaStream_t)stream)));
  return TYLO_OK;
}

extern "C" int32_t tylo_b200_distill_bwd(void* dX, const float* dLoss, const void* X, const float* teacher, const int32_t* index,
                                         const float* Mx, const float* L, int32_t K, int64_t M, int64_t N, int64_t ldx,
                                         float temperature, float teacher_temperature, int32_t renormalize, int32_t dtype,
                                         tylo_stream_t stream) {
  const char* who = "distill_bwd";
  if (int32_t rc = check_distill(who, X, teacher, index, K, M, N, ldx, temperature, teacher_temperature)) return rc;
  if (int32_t rc = check_vocab_grad(who, dX, X, M, N, ldx, dtype)) return rc;
  TYLO_REQUIRE(dLoss, TYLO_ERR_INVALID_ARGUMENT, "%s: dLoss must be non-null", who);
  TYLO_REQUIRE(Mx && L, TYLO_ERR_INVALID_ARGUMENT, "%s: checkpoints Mx and L from the forward are required", who);
  DistillArgs a = distill_args(X, teacher, index, K, M, ldx, temperature, teacher_temperature, renormalize);
  a.dX = dX; a.dLoss = dLoss; a.inMx = Mx; a.inL = L;
  TYLO_DISPATCH_DTYPE(dtype, T, return (distill_dispatch<T, false, true>(who, a, N, (cudaStream_t)stream)));
  return TYLO_OK;
}

extern "C" int32_t tylo_b200_distill_fwd_bwd(float* Loss, void* dX, const float* dLoss, const void* X, const float* teacher,
                                             const int32_t* index, int32_t K, int64_t M, int64_t N, int64_t ldx, float temperature,
                                             float teacher_temperature, int32_t renormalize, int32_t dtype, tylo_stream_t stream) {
  const char* who = "distill_fwd_bwd";
  if (int32_t rc = check_distill(who, X, teacher, index, K, M, N, ldx, temperature, teacher_temperature)) return rc;
  if (int32_t rc = check_vocab_grad(who, dX, X, M, N, ldx, dtype)) return rc;
  TYLO_REQUIRE(Loss && dLoss, TYLO_ERR_INVALID_ARGUMENT, "%s: Loss and dLoss must be non-null", who);
  TYLO_REQUIRE(Loss != dLoss, TYLO_ERR_INVALID_ARGUMENT, "%s: Loss and dLoss must be different arrays", who);
  DistillArgs a = distill_args(X, teacher, index, K, M, ldx, temperature, teacher_temperature, renormalize);
  a.Loss = Loss; a.dX = dX; a.dLoss = dLoss;
  TYLO_DISPATCH_DTYPE(dtype, T, return (distill_dispatch<T, true, true>(who, a, N, (cudaStream_t)stream)));
  return TYLO_OK;
}
