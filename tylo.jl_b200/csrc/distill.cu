// Distillation from a teacher's top logits, and its gradient.  With q = softmax(x / t) of the student's row and the teacher's K
// entries (value v_k at index I_k, temperature u), p_k = exp(v_k / u) / sum_j exp(v_j / u), or exp(v_k / u) as it is where the
// teacher's own mass is kept:
//
//   loss = sum_k p_k (log p_k - log q_{I_k})
//   dX_j = w / t (P q_j - sum_{k: I_k = j} p_k),   P = sum_k p_k
//
// Entries with an index outside [0, M) are left out, of the teacher's normalisation too.
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
  int M, K, renormalize;
  float temperature, teacher_temperature;
};

// Places for K entries in each of the three arrays, so that what follows them is 16-byte aligned.
__host__ __device__ constexpr int entry_slots(int K) { return (K + 3) / 4 * 4; }

// The teacher's probabilities of a row into shared memory (-1 as the index of an entry that is left out); returns the normaliser's
// logarithm, so that log p_k = v_k / u - the result, and P through `mass`.
template <int THREADS>
__device__ __forceinline__ float teacher_row(const DistillArgs& a, size_t row, float* p, int* index, float* scratch, float& mass) {
  const float* v = a.teacher + row * a.K;
  const int32_t* id = a.index + row * a.K;
  float m = -INFINITY;
  for (int k = threadIdx.x; k < a.K; k += THREADS) {
    const int j = id[k];
    const bool live = j >= 0 && j < a.M;
    const float z = live ? v[k] / a.teacher_temperature : -INFINITY;
    index[k] = live ? j : -1;
    p[k] = z;
    m = fmaxf(m, z);
  }
  float log_norm = 0.f;
  if (a.renormalize) {
    m = block_reduce<THREADS>(m, MaxOp(), -INFINITY, scratch);
    const float mo = m == -INFINITY ? 0.f : m;
    float s = 0.f;
    for (int k = threadIdx.x; k < a.K; k += THREADS) s += expf(p[k] - mo);
    s = block_reduce<THREADS>(s, SumOp(), 0.f, scratch);
    log_norm = s == 0.f ? 0.f : mo + logf(s);
  }
  float sum = 0.f;
  for (int k = threadIdx.x; k < a.K; k += THREADS) {
    p[k] = expf(p[k] - log_norm);
    sum += p[k];
  }
  mass = block_reduce<THREADS>(sum, SumOp(), 0.f, scratch);     // its barriers also publish p and index
  return log_norm;
}

// GROUPS > 0: the part waits in shared memory for the second look.  Dynamic shared memory: the teacher's entries, then the part.
template <typename T, int THREADS, int U, int GROUPS, bool LOSS, bool GRAD>
__global__ void __launch_bounds__(THREADS, THREADS == 128 ? 8 : THREADS == 256 ? 5 : GROUPS ? 2 : GRAD ? 3 : 4)
distill_row_kernel(const DistillArgs a, int parts) {
  __shared__ float scratch[100];
  extern __shared__ uint4 dynamic[];
  const int slots = entry_slots(a.K);
  float *p = reinterpret_cast<float*>(dynamic), *xk = p + slots;
  int* index = reinterpret_cast<int*>(xk + slots);
  uint4* kept = reinterpret_cast<uint4*>(index + slots);
  const size_t row = blockIdx.x / parts;
  const T* x = (const T*)a.X + row * a.ldx;
  const VocabRow<T> r(x, a.M);
  const VocabPart part(blockIdx.x % parts, parts, r.whole);
  const float it = 1.f / a.temperature, scale = kVocabLog2e / a.temperature;
  VocabStats st;
  if constexpr (GROUPS > 0) st = vocab_resident_stats<T, THREADS, U, GROUPS, false>(kept, x, r, part, scale);
  else if constexpr (LOSS) st = vocab_thread_stats<T, THREADS, U, false, GRAD, false>(x, r, part, scale, nullptr);
  float mass;
  const float log_norm = teacher_row<THREADS>(a, row, p, index, scratch, mass);
  for (int k = threadIdx.x; k < a.K; k += THREADS) xk[k] = index[k] >= 0 ? Elem<T>::to_f(x[index[k]]) : 0.f;
  if constexpr (LOSS) vocab_reduce<THREADS, false>(st, scale, scratch, parts);
  else st = {a.inMx[row], 0.f, a.inL[row], 0.f};
  const float mo = st.m == -INFINITY ? 0.f : st.m;
  if (LOSS && part.part == 0) {
    const float logL = st.s == 0.f ? 0.f : logf(st.s);
    float loss = 0.f;
    for (int k = threadIdx.x; k < a.K; k += THREADS)
      if (index[k] >= 0 && p[k] != 0.f)
        loss += p[k] * ((a.teacher[row * a.K + k] / a.teacher_temperature - log_norm) - ((xk[k] - mo) / a.temperature - logL));
    loss = block_reduce<THREADS>(loss, SumOp(), 0.f, scratch);
    if (threadIdx.x == 0) {
      a.Loss[row] = loss;
      if (a.Mx) { a.Mx[row] = st.m; a.L[row] = st.s; }
    }
  }
  if constexpr (GRAD) {
    T* dx = (T*)a.dX + row * a.ldx;
    const float w = a.dLoss[row] * it;
    if (w == 0.f || mass == 0.f || st.s == 0.f) {       // no weight, no teacher or no probability anywhere
      vocab_zero<T, THREADS>(dx, r, part);
    } else {
      const float2 m2 = make_float2(-mo, -mo), sc = make_float2(scale, scale), c = make_float2(w * mass / st.s, w * mass / st.s);
      auto grad = [&](float2 f) {
        const float2 y = __fmul2_rn(__fadd2_rn(f, m2), sc);
        return __fmul2_rn(make_float2(vocab_ex2(y.x), vocab_ex2(y.y)), c);
      };
      if (!LOSS) __syncthreads();             // xk is read before any gradient is written: dX may be X
      if constexpr (GROUPS > 0) vocab_resident_rewrite<T, THREADS, U>(dx, kept, x, r, part, grad);
      else vocab_rewrite<T, THREADS, U>(dx, x, r, part, grad);
      __syncthreads();
      // the teacher's entries in this part: every copy of an index sums all its copies in the same order and stores the same value
      for (int k = threadIdx.x; k < a.K; k += THREADS) {
        const int j = index[k];
        if (j < 0 || part.template owner<THREADS>(r, j) < 0) continue;
        float sum = 0.f;
        for (int i = 0; i < a.K; ++i) sum += index[i] == j ? p[i] : 0.f;
        dx[j] = Elem<T>::from_f(grad(make_float2(xk[k], 0.f)).x - w * sum);
      }
    }
  }
  if constexpr (LOSS) cluster_done(parts);
}

template <typename T, bool LOSS, bool GRAD>
static int32_t distill_dispatch(const char* who, const DistillArgs& a, int64_t N, cudaStream_t stream) {
  const int64_t packets = a.M / Elem<T>::kVec;
  const int entries = 12 * entry_slots(a.K);
  if constexpr (!LOSS) {       // nothing to tell one another: plain CTAs, as many per row as fill the GPU several times over
    int parts = 1;
    while (parts < 64 && N * parts < 16 * sm_count() && packets >= 8LL * parts * 512) parts *= 2;
    if (packets <= 1024) distill_row_kernel<T, 128, 4, 0, LOSS, GRAD><<<(unsigned)N, 128, entries, stream>>>(a, 1);
    else distill_row_kernel<T, 512, 4, 0, LOSS, GRAD><<<(unsigned)(N * parts), 512, entries, stream>>>(a, parts);
    return check_launch(who);
  } else {
    const int parts = vocab_parts(N, packets);
    if constexpr (!GRAD) {
      if (packets <= 1024) return launch_vocab(who, distill_row_kernel<T, 128, 4, 0, LOSS, GRAD>, a, N, parts, 128, stream, entries);
      return launch_vocab(who, distill_row_kernel<T, 512, 4, 0, LOSS, GRAD>, a, N, parts, 512, stream, entries);
    } else {
      const int64_t per = (packets + parts - 1) / parts;
#define TYLO_BOTH(THREADS, U, GROUPS) \
  launch_vocab(who, distill_row_kernel<T, THREADS, U, GROUPS, LOSS, GRAD>, a, N, parts, THREADS, stream, entries + (GROUPS ? (int)per * 16 : 0))
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
  a.X = X; a.teacher = teacher; a.index = index; a.K = K; a.M = (int)M; a.ldx = ldx;
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
  TYLO_REQUIRE(dX && dLoss, TYLO_ERR_INVALID_ARGUMENT, "%s: dX and dLoss must be non-null", who);
  TYLO_REQUIRE(aligned16(dX), TYLO_ERR_MISALIGNED, "%s: dX must be 16-byte aligned", who);
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
  TYLO_REQUIRE(Loss && dX && dLoss, TYLO_ERR_INVALID_ARGUMENT, "%s: Loss, dX and dLoss must be non-null", who);
  TYLO_REQUIRE(aligned16(dX), TYLO_ERR_MISALIGNED, "%s: dX must be 16-byte aligned", who);
  DistillArgs a = distill_args(X, teacher, index, K, M, ldx, temperature, teacher_temperature, renormalize);
  a.Loss = Loss; a.dX = dX; a.dLoss = dLoss;
  TYLO_DISPATCH_DTYPE(dtype, T, return (distill_dispatch<T, true, true>(who, a, N, (cudaStream_t)stream)));
  return TYLO_OK;
}
