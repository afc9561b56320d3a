// Log probabilities of given tokens with the row's entropy and its largest alternatives, and their gradient.
//
//   logp = y_target - log L,   H = log L - A / L,   A = sum exp(y) y                      (y, L as in vocab.cuh)
//   dX_j = 1/t ( g ([j = target] - p_j) - h p_j (log p_j + H) )
#include "vocab.cuh"

namespace tylo {

struct LogprobArgs {
  const void* X;
  const int32_t* targets;
  float *Logp, *Entropy, *TopLogp, *Mx, *L;
  int32_t* TopIndex;
  void* dX;
  const float *dLogp, *dEntropy;
  const float *inEntropy, *inMx, *inL;
  int64_t ldx;
  int M, top;
  float temperature;
};

constexpr int kLogprobThreads = 512;

__device__ __forceinline__ uint64_t block_max_key(uint64_t k, uint64_t* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t k2 = __shfl_xor_sync(0xffffffffu, k, o);
    k = k2 > k ? k2 : k;
  }
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = k;
  __syncthreads();
  k = 0;
  for (int w = 0; w < kLogprobThreads / 32; ++w) k = scratch[w] > k ? scratch[w] : k;
  __syncthreads();
  return k;
}

// Writes the gradient of a row: p (c0 + c1 log2 p) per element, c0 = -(g + h H) / t, c1 = -h ln 2 / t, and g / t at the target.
template <typename T>
__device__ __forceinline__ void logprob_row_grad(T* dx, const T* x, const VocabRow<T>& r, int first, int step, int last, bool singles,
                                                 int target, float mx, float L, float g, float h, float H, float temperature) {
  constexpr int VEC = Elem<T>::kVec;
  const float it = 1.f / temperature, scale = kVocabLog2e * it;
  const bool none = (g == 0.f && h == 0.f) || L == 0.f;
  const float mo = mx == -INFINITY ? 0.f : mx, inv = 1.f / L, lg = log2f(L);
  const float c0 = -(h == 0.f ? g : g + h * H) * it, c1 = -h * kVocabLn2 * it, at = g * it;
  auto grad = [&](float f, int j) {
    const float y = (f - mo) * scale, p = vocab_ex2(y) * inv;
    float d = p * fmaf(c1, fmaxf(y, kExpFloor) - lg, c0);
    if (j == target) d += at;
    return none ? 0.f : d;
  };
  const int one = r.single(threadIdx.x);
  if (singles && one >= 0) dx[one] = Elem<T>::from_f(grad(Elem<T>::to_f(x[one]), one));
  for (int v = first; v < last; v += step) {
    Pack<T> p;
    p.raw = ld_logits(x + r.index(v));
    float f[VEC];
    p.unpack(f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = grad(f[j], r.index(v) + j);
    p.pack(f);
    st_stream(dx + r.index(v), p.raw);
  }
}

template <typename T, bool ENTROPY, bool GRAD>
__global__ void __launch_bounds__(kLogprobThreads) logprob_row_kernel(const LogprobArgs a) {
  constexpr int VEC = Elem<T>::kVec;
  __shared__ float scratch[100];
  __shared__ uint64_t keys[32];
  const size_t row = blockIdx.x;
  const T* x = (const T*)a.X + row * a.ldx;
  const VocabRow<T> r(x, a.M);
  const float scale = kVocabLog2e / a.temperature;
  const int target = a.targets ? a.targets[row] : -1;
  const bool has = target >= 0 && target < a.M;
  const float xt = has ? Elem<T>::to_f(x[target]) : 0.f;
  VocabStats st = vocab_thread_stats<T, kLogprobThreads, 4, ENTROPY>(x, r, VocabPart(0, 1, r.whole), scale);
  vocab_reduce<kLogprobThreads>(st, scale, scratch, 1);
  const float logL = st.s == 0.f ? 0.f : logf(st.s), H = st.s == 0.f ? 0.f : logL - kVocabLn2 * st.a / st.s;
  const float mo = st.m == -INFINITY ? 0.f : st.m;
  if (threadIdx.x == 0) {
    if (a.Logp) a.Logp[row] = has ? (xt - mo) / a.temperature - logL : 0.f;
    if (a.Entropy) a.Entropy[row] = H;
    if (a.Mx) { a.Mx[row] = st.m; a.L[row] = st.s; }
  }
  uint64_t below = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t best = 0;
    const int one = r.single(threadIdx.x);
    if (one >= 0) {
      const uint64_t key = vocab_key(Elem<T>::to_f(x[one]), one);
      if (key < below) best = key;
    }
    for (int v = threadIdx.x; v < r.whole; v += kLogprobThreads) {
      Pack<T> p;
      p.raw = ld_logits(x + r.index(v));
      float f[VEC];
      p.unpack(f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const uint64_t key = vocab_key(f[j], r.index(v) + j);
        if (key < below && key > best) best = key;
      }
    }
    below = block_max_key(best, keys);
    if (threadIdx.x == 0) {
      a.TopLogp[row * a.top + k] = (vocab_unkey((uint32_t)(below >> 32)) - mo) / a.temperature - logL;
      a.TopIndex[row * a.top + k] = vocab_key_index(below);
    }
  }
  if constexpr (GRAD)
    logprob_row_grad<T>((T*)a.dX + row * a.ldx, x, r, threadIdx.x, kLogprobThreads, r.whole, true, has ? target : -1, st.m, st.s,
                        has ? a.dLogp[row] : 0.f, a.dEntropy ? a.dEntropy[row] : 0.f, H, a.temperature);
}

template <typename T>
__global__ void __launch_bounds__(kLogprobThreads) logprob_bwd_kernel(const LogprobArgs a) {
  const size_t row = blockIdx.x;
  const T* x = (const T*)a.X + row * a.ldx;
  const VocabRow<T> r(x, a.M);
  const int target = a.targets ? a.targets[row] : -1;
  const bool has = target >= 0 && target < a.M;
  logprob_row_grad<T>((T*)a.dX + row * a.ldx, x, r, threadIdx.x, kLogprobThreads, r.whole, true, has ? target : -1, a.inMx[row], a.inL[row],
                      has ? a.dLogp[row] : 0.f, a.dEntropy ? a.dEntropy[row] : 0.f, a.dEntropy ? a.inEntropy[row] : 0.f, a.temperature);
}

}  // namespace tylo

using namespace tylo;

extern "C" int32_t tylo_b200_token_logprobs_fwd(float* Logp, float* Entropy, float* TopLogp, int32_t* TopIndex, float* Mx, float* L,
                                                const void* X, const int32_t* targets, int32_t top, int64_t M, int64_t N,
                                                int64_t ldx, float temperature, int32_t dtype, tylo_stream_t stream) {
  const char* who = "token_logprobs_fwd";
  if (int32_t rc = check_vocab(who, X, M, N, ldx, temperature)) return rc;
  TYLO_REQUIRE(Logp || Entropy || TopLogp || Mx, TYLO_ERR_INVALID_ARGUMENT, "%s: nothing to compute", who);
  TYLO_REQUIRE(!Logp == !targets, TYLO_ERR_INVALID_ARGUMENT, "%s: Logp and targets go together", who);
  TYLO_REQUIRE(!Mx == !L, TYLO_ERR_INVALID_ARGUMENT, "%s: checkpoints Mx and L go together", who);
  TYLO_REQUIRE(top >= 0 && top <= TYLO_TOP_MAX && top <= M, TYLO_ERR_INVALID_ARGUMENT,
               "%s: top (%d) must be between 0 and %d and at most M (%lld)", who, top, TYLO_TOP_MAX, (long long)M);
  TYLO_REQUIRE((top > 0) == (TopLogp != nullptr) && (top > 0) == (TopIndex != nullptr), TYLO_ERR_INVALID_ARGUMENT,
               "%s: TopLogp and TopIndex go with top > 0", who);
  LogprobArgs a = {};
  a.X = X; a.targets = targets; a.Logp = Logp; a.Entropy = Entropy; a.TopLogp = TopLogp; a.TopIndex = TopIndex; a.Mx = Mx; a.L = L;
  a.ldx = ldx; a.M = (int)M; a.top = top; a.temperature = temperature;
  TYLO_DISPATCH_DTYPE(dtype, T, {
    if (Entropy) logprob_row_kernel<T, true, false><<<(unsigned)N, kLogprobThreads, 0, (cudaStream_t)stream>>>(a);
    else logprob_row_kernel<T, false, false><<<(unsigned)N, kLogprobThreads, 0, (cudaStream_t)stream>>>(a);
  });
  return check_launch(who);
}

static int32_t check_logprob_grad(const char* who, const void* dX, const float* dLogp, const float* dEntropy, const int32_t* targets) {
  TYLO_REQUIRE(dX, TYLO_ERR_INVALID_ARGUMENT, "%s: dX must be non-null", who);
  TYLO_REQUIRE(aligned16(dX), TYLO_ERR_MISALIGNED, "%s: dX must be 16-byte aligned", who);
  TYLO_REQUIRE(!dLogp == !targets, TYLO_ERR_INVALID_ARGUMENT, "%s: dLogp and targets go together", who);
  TYLO_REQUIRE(dLogp || dEntropy, TYLO_ERR_INVALID_ARGUMENT, "%s: dLogp or dEntropy is required", who);
  return TYLO_OK;
}

extern "C" int32_t tylo_b200_token_logprobs_bwd(void* dX, const float* dLogp, const float* dEntropy, const void* X,
                                                const int32_t* targets, const float* Entropy, const float* Mx, const float* L,
                                                int64_t M, int64_t N, int64_t ldx, float temperature, int32_t dtype,
                                                tylo_stream_t stream) {
  const char* who = "token_logprobs_bwd";
  if (int32_t rc = check_vocab(who, X, M, N, ldx, temperature)) return rc;
  if (int32_t rc = check_logprob_grad(who, dX, dLogp, dEntropy, targets)) return rc;
  TYLO_REQUIRE(Mx && L, TYLO_ERR_INVALID_ARGUMENT, "%s: checkpoints Mx and L from the forward are required", who);
  TYLO_REQUIRE(!dEntropy || Entropy, TYLO_ERR_INVALID_ARGUMENT, "%s: dEntropy needs the forward's Entropy", who);
  LogprobArgs a = {};
  a.X = X; a.targets = targets; a.dX = dX; a.dLogp = dLogp; a.dEntropy = dEntropy; a.inEntropy = Entropy; a.inMx = Mx; a.inL = L;
  a.ldx = ldx; a.M = (int)M; a.temperature = temperature;
  TYLO_DISPATCH_DTYPE(dtype, T, (logprob_bwd_kernel<T><<<(unsigned)N, kLogprobThreads, 0, (cudaStream_t)stream>>>(a)));
  return check_launch(who);
}

extern "C" int32_t tylo_b200_token_logprobs_fwd_bwd(float* Logp, float* Entropy, void* dX, const float* dLogp, const float* dEntropy,
                                                    const void* X, const int32_t* targets, int64_t M, int64_t N, int64_t ldx,
                                                    float temperature, int32_t dtype, tylo_stream_t stream) {
  const char* who = "token_logprobs_fwd_bwd";
  if (int32_t rc = check_vocab(who, X, M, N, ldx, temperature)) return rc;
  if (int32_t rc = check_logprob_grad(who, dX, dLogp, dEntropy, targets)) return rc;
  TYLO_REQUIRE(!Logp || targets, TYLO_ERR_INVALID_ARGUMENT, "%s: Logp needs targets", who);
  LogprobArgs a = {};
  a.X = X; a.targets = targets; a.Logp = Logp; a.Entropy = Entropy; a.dX = dX; a.dLogp = dLogp; a.dEntropy = dEntropy;
  a.ldx = ldx; a.M = (int)M; a.temperature = temperature;
  TYLO_DISPATCH_DTYPE(dtype, T, {
    if (Entropy || dEntropy) logprob_row_kernel<T, true, true><<<(unsigned)N, kLogprobThreads, 0, (cudaStream_t)stream>>>(a);
    else logprob_row_kernel<T, false, true><<<(unsigned)N, kLogprobThreads, 0, (cudaStream_t)stream>>>(a);
  });
  return check_launch(who);
}
