// Log probabilities of given tokens with the row's entropy and its largest alternatives, and their gradient.
//
//   logp = y_target - log L,   H = log L - A / L,   A = sum exp(y) y                      (y, L as in vocab.cuh)
//   dX_j = 1/t ( g ([j = target] - p_j) - h p_j (log p_j + H) )
//
// Times are us of a pass among others in runs of a second and more, where the card is at its power cap; short runs take up to a tenth less,
// cards differ by a twentieth.  bf16 unless said otherwise.
// Forward: one pass over the row, which memory bounds: 2048 x 131072 86 to 90 = 6.2 TB/s (a plain read of the same bytes takes 76 in short
// runs, this 79), fp16 91, 1024 x 131072 fp32 80; with the entropy 4096 x 65536 99.  The special-function units, one exponential per logit,
// are three quarters busy beside it.  Smaller CTAs for shorter rows, so that starting a CTA and joining its sums weigh less: 4096 x 32768 46
// to 49 with 256 threads, 8192 x 16000 50 with 128 (67 with 512 when that was chosen).  Below that the CTA a row costs more than the row:
// 8192 x 4000 19 for 10 us of bytes, 8192 x 1000 16 for 2.5.
// Alternatives: what follows the sums is a chain of short steps, hidden by the other CTAs of the SM only.
//   alternatives      0    20   128   256                            0    20    64   128   256
//   2048 x 131072    86   103   122   157      8192 x 4000           19    50    64   117   293
//   4096 x 32768     46    65    94   168      8192 x 1000           16    47    64   211   365
//   8192 x 16000     49    78   139   287      8192 x 1100, 150: 511 (the bound is below every element, and raised)
// A mask that leaves 40: 256 x 32000 fp16 with 64 of them 13.2 and 16.4 masked, with 200 16.4 and 20.6; 3000 x 1000 with 100 58 and 165, with
// 256 141 and 262.
// Backward: one read and one write, 4096 x 65536 160 = 6.7 TB/s, with the entropy's weight 171.
// Value and gradient in one launch read the logits from memory once: 4096 x 32768 104 to 107 = 5.1 TB/s, with the entropy 113, fp16 105, 2048 x
// 32768 fp32 96, the two calls with the entropy 139; 8192 x 16000 103.  The second look finds two thirds of a longer row in L2: 2048 x 131072
// 210, 1024 x 131072 fp32 217, 2048 x 262144 431.  Rows whose target is no token are read all the same: half of them such, 99 and 195.
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
  int M, top, sms;
  float temperature;
};

__device__ __forceinline__ float vocab_logp(float x, const VocabStats& st, float temperature) {
  return (x - (st.m == -INFINITY ? 0.f : st.m)) / temperature - (st.s == 0.f ? 0.f : logf(st.s));
}
__device__ __forceinline__ float vocab_entropy(const VocabStats& st) {
  return st.s == 0.f ? 0.f : logf(st.s) - kVocabLn2 * st.a / st.s;
}

// A row's gradient: dX_j = e_j (A y_j + B) with e_j = exp2(y_j), y_j in units of log 2, and `at` added at the target.
template <bool ENTROPY> struct LogprobGrad {
  float2 mo, scale, A, B;
  float at;
  __device__ __forceinline__ LogprobGrad(float mx, float L, float g, float h, float H, float temperature) {
    const float it = 1.f / temperature, c = it / L, m = mx == -INFINITY ? 0.f : -mx, k = kVocabLog2e / temperature;
    // -p (g + h (log p + H)) / t with log p = ln 2 (y - log2 L)
    const float a = -h * kVocabLn2 * c, b = -(ENTROPY ? g + h * (H - logf(L)) : g) * c;
    mo = make_float2(m, m); scale = make_float2(k, k); A = make_float2(a, a); B = make_float2(b, b);
    at = g * it;
  }
  __device__ __forceinline__ float2 operator()(float2 x) const {
    const float2 y = __fmul2_rn(__fadd2_rn(x, mo), scale);
    const float2 e = make_float2(vocab_ex2(y.x), vocab_ex2(y.y));
    if constexpr (ENTROPY) return __fmul2_rn(e, __ffma2_rn(A, make_float2(fmaxf(y.x, kExpFloor), fmaxf(y.y, kExpFloor)), B));
    else return __fmul2_rn(e, B);
  }
};

// The gradient of a part, which waits in `kept` or, without that, is read (again).  `xt`: the target's logit, read before anything is written (dX may
// be X); target < 0: none.  A row without weights or without any probability gets zeros.
template <typename T, int THREADS, int U, bool ENTROPY>
__device__ __forceinline__ void logprob_part_grad(const LogprobArgs& a, size_t row, const T* x, const uint4* kept, const VocabRow<T>& r,
                                                  const VocabPart& part, int target, float xt, float mx, float L, float g, float h, float H) {
  T* dx = (T*)a.dX + row * a.ldx;
  if ((g == 0.f && h == 0.f) || L == 0.f) {
    vocab_zero<T, THREADS>(dx, r, part);
    return;
  }
  const LogprobGrad<ENTROPY> d(mx, L, g, h, H, a.temperature);
  if (kept) vocab_resident_rewrite<T, THREADS, U>(dx, kept, x, r, part, d);
  else vocab_rewrite<T, THREADS, U>(dx, x, r, part, d);
  if (target >= 0 && part.template owner<THREADS>(r, target) == (int)threadIdx.x) dx[target] = Elem<T>::from_f(d(make_float2(xt, 0.f)).x + d.at);
}

// CTAs per SM: registers for as many as the loads need to be hidden behind one another.  With alternatives five of 256 threads, three of
// 512: 2048 x 131072, 20 of them 107 us with five, 111 with six, 115 with four.
constexpr int logprob_ctas(int threads, bool entropy, bool top) {
  return top ? (threads == 128 ? 8 : threads == 256 ? 5 : 3) : 512 / threads * (entropy ? 3 : 4);
}

template <typename T, int THREADS, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(THREADS, logprob_ctas(THREADS, ENTROPY, TOP)) logprob_fwd_kernel(const LogprobArgs a, int parts) {
  __shared__ float scratch[100];
  const size_t row = blockIdx.x / parts;
  const T* x = (const T*)a.X + row * a.ldx;
  const VocabRow<T> r(x, a.M);
  const VocabPart part(blockIdx.x % parts, parts, r.whole);
  const float scale = kVocabLog2e / a.temperature;
  const bool lead = threadIdx.x == 0 && part.part == 0;
  const int target = lead && a.Logp ? a.targets[row] : -1;       // (first used behind the sums: nothing waits for it here)
  extern __shared__ uint64_t top_space[];
  TopScratch<THREADS>& top = *reinterpret_cast<TopScratch<THREADS>*>(top_space);
  const VocabCells<THREADS> cells(TOP ? top.cells : nullptr, part.hi - part.lo, 4 * THREADS);
  VocabStats st = vocab_thread_stats<T, THREADS, 4, ENTROPY, false, TOP>(x, r, part, scale, &cells);
  const bool has = target >= 0 && target < a.M;
  const float xt = has ? Elem<T>::to_f(x[target]) : 0.f;
  vocab_ask_ahead((const T*)a.X, a.ldx, a.M, row, a.sms * logprob_ctas(THREADS, ENTROPY, TOP), parts);
  const bool odd = st.s != st.s;
  if constexpr (TOP) top.mine[threadIdx.x] = vocab_mine<T, THREADS>(x, r, part, st);
  vocab_reduce<THREADS, ENTROPY>(st, scale, scratch, parts);
  if (lead) {
    if (a.Logp) a.Logp[row] = has ? vocab_logp(xt, st, a.temperature) : 0.f;
    if (a.Entropy) a.Entropy[row] = vocab_entropy(st);
    if (a.Mx) { a.Mx[row] = st.m; a.L[row] = st.s; }
  }
  if constexpr (TOP) {
    const int n = vocab_top<T, THREADS, 4>(x, r, part, a.top, cells, odd, top);
    vocab_ranked<THREADS>(top, n, a.top, parts, [&](int rank, uint64_t key) {
      a.TopLogp[row * a.top + rank] = vocab_logp(vocab_unkey((uint32_t)(key >> 32)), st, a.temperature);
      a.TopIndex[row * a.top + rank] = vocab_key_index(key);
    });
  }
  cluster_done(parts);
}

// Value and gradient.  GROUPS > 0: the part waits in shared memory for the second look; 0: it is too long for that and is read again, out of
// L2 as far as it is still there (both sides: TYLO_VOCAB_RESIDENT).
template <typename T, int THREADS, int U, int GROUPS, bool ENTROPY>
__global__ void __launch_bounds__(THREADS, THREADS == 128 ? 8 : THREADS == 256 ? 5 : GROUPS ? 2 : 3)
logprob_fwd_bwd_kernel(const LogprobArgs a, int parts) {
  extern __shared__ uint4 kept[];
  __shared__ float scratch[100];
  const size_t row = blockIdx.x / parts;
  const T* x = (const T*)a.X + row * a.ldx;
  const VocabRow<T> r(x, a.M);
  const VocabPart part(blockIdx.x % parts, parts, r.whole);
  const float scale = kVocabLog2e / a.temperature;
  const int target = a.targets ? a.targets[row] : -1;            // (first used behind the sums: nothing waits for these here)
  float g = a.targets ? a.dLogp[row] : 0.f;
  const float h = ENTROPY && a.dEntropy ? a.dEntropy[row] : 0.f;
  VocabStats st;
  if constexpr (GROUPS > 0) {
    vocab_resident_ask<T, THREADS, U, GROUPS>(kept, x, r, part);
    st = vocab_resident_stats<T, THREADS, U, GROUPS, ENTROPY>(kept, x, r, part, scale);
  } else st = vocab_thread_stats<T, THREADS, U, ENTROPY, true, false>(x, r, part, scale, nullptr);
  const bool has = target >= 0 && target < a.M;
  const float xt = has ? Elem<T>::to_f(x[target]) : 0.f;
  g = has ? g : 0.f;
  vocab_reduce<THREADS, ENTROPY>(st, scale, scratch, parts);
  float H = 0.f;
  if constexpr (ENTROPY) H = vocab_entropy(st);
  if (threadIdx.x == 0 && part.part == 0) {
    if (a.Logp) a.Logp[row] = has ? vocab_logp(xt, st, a.temperature) : 0.f;
    if (a.Entropy) a.Entropy[row] = H;
  }
  logprob_part_grad<T, THREADS, U, ENTROPY>(a, row, x, GROUPS > 0 ? kept : nullptr, r, part, has ? target : -1, xt, st.m, st.s, g, h, H);
  cluster_done(parts);
}

// 2,048 packets per CTA: a row's coefficients cost a thread as much as three packets (1,024: 4096 x 65536 bf16 with both weights 200 us,
// 161 with 2,048).  From the last row to the first: what the forward read last is still in L2 (forward and backward, 4096 x 32768 bf16 133
// and 128.5 us, 777 x 50001 fp32 83.3 and 81.6, 4096 x 65536 259.9 and 256.4).
template <typename T, int THREADS, bool ENTROPY>
__global__ void __launch_bounds__(THREADS, 6) logprob_bwd_kernel(const LogprobArgs a, int parts) {
  const size_t row = (gridDim.x - 1 - blockIdx.x) / parts;
  const T* x = (const T*)a.X + row * a.ldx;
  const VocabRow<T> r(x, a.M);
  const VocabPart part((gridDim.x - 1 - blockIdx.x) % parts, parts, r.whole);
  const int target = a.targets ? a.targets[row] : -1;
  const bool has = target >= 0 && target < a.M;
  const float xt = has ? Elem<T>::to_f(x[target]) : 0.f;
  // (in place: the thread that uses xt is the one that writes its packet, later)
  logprob_part_grad<T, THREADS, 4, ENTROPY>(a, row, x, nullptr, r, part, has ? target : -1, xt, a.inMx[row], a.inL[row], has ? a.dLogp[row] : 0.f,
                                         ENTROPY ? a.dEntropy[row] : 0.f, ENTROPY ? a.inEntropy[row] : 0.f);
}

template <typename T, bool ENTROPY>
static int32_t logprob_fwd_dispatch(const char* who, const LogprobArgs& a, int64_t N, cudaStream_t stream) {
  const int64_t packets = a.M / Elem<T>::kVec;
  const int parts = vocab_parts(N, packets);
  const int64_t per = (packets + parts - 1) / parts;
  // us, bf16.  256 threads up to 176 alternatives (256 / 512 threads: 4096 x 32768 with 144 of them 105 / 132, with 200 136 / 143; 2048 x
  // 131072 129 / 133 and 147 / 142): with more, the threads' maxima bound too little.  128 for a clustered row, whose lists have to fit
  // into 4 * THREADS places.  128 threads for many short rows (256 / 128: 8192 x 16000 with 20 108 / 81, 4096 x 32768 78 / 71, 2048 x 131072
  // with 64 115 / 123, 256 x 32000 13.2 / 15.6).  The rule was found on rows of 16,000 logits and more.
#define TYLO_TOP(THREADS) \
  launch_vocab(who, logprob_fwd_kernel<T, THREADS, ENTROPY, true>, a, N, parts, THREADS, stream, (int)sizeof(TopScratch<THREADS>))
  if (a.top && a.top <= 64 && per <= 4096 && N * parts >= 8 * sm_count()) return TYLO_TOP(128);
  if (a.top) return a.top <= (parts == 1 ? 176 : 128) ? TYLO_TOP(256) : TYLO_TOP(512);
#undef TYLO_TOP
#define TYLO_FWD(THREADS) launch_vocab(who, logprob_fwd_kernel<T, THREADS, ENTROPY, false>, a, N, parts, THREADS, stream)
  TYLO_VOCAB_STREAM(TYLO_FWD);
#undef TYLO_FWD
}

template <typename T, bool ENTROPY>
static int32_t logprob_fwd_bwd_dispatch(const char* who, const LogprobArgs& a, int64_t N, cudaStream_t stream) {
  const int64_t packets = a.M / Elem<T>::kVec;
  const int parts = vocab_parts_twice(N, packets, 14336);
  const int64_t per = (packets + parts - 1) / parts;
#define TYLO_BOTH(THREADS, U, GROUPS) \
  launch_vocab(who, logprob_fwd_bwd_kernel<T, THREADS, U, GROUPS, ENTROPY>, a, N, parts, THREADS, stream, GROUPS ? (int)per * 16 : 0)
  TYLO_VOCAB_RESIDENT(TYLO_BOTH);
#undef TYLO_BOTH
}

template <typename T>
static int32_t logprob_bwd_dispatch(const char* who, const LogprobArgs& a, int64_t N, cudaStream_t stream) {
  constexpr int THREADS = 256;
  const int64_t packets = a.M / Elem<T>::kVec;
  const int parts = (int)((packets + 8 * THREADS - 1) / (8 * THREADS) + (packets == 0));
  if (a.dEntropy) logprob_bwd_kernel<T, THREADS, true><<<(unsigned)(N * parts), THREADS, 0, stream>>>(a, parts);
  else logprob_bwd_kernel<T, THREADS, false><<<(unsigned)(N * parts), THREADS, 0, stream>>>(a, parts);
  return check_launch(who);
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
  a.ldx = ldx; a.M = (int)M; a.top = top; a.sms = sm_count(); a.temperature = temperature;
  TYLO_DISPATCH_DTYPE(dtype, T, return (Entropy ? logprob_fwd_dispatch<T, true>(who, a, N, (cudaStream_t)stream)
                                                : logprob_fwd_dispatch<T, false>(who, a, N, (cudaStream_t)stream)));
  return TYLO_OK;
}

static int32_t check_logprob_weights(const char* who, const float* dLogp, const float* dEntropy, const int32_t* targets) {
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
  if (int32_t rc = check_vocab_grad(who, dX, X, M, N, ldx, dtype)) return rc;
  if (int32_t rc = check_logprob_weights(who, dLogp, dEntropy, targets)) return rc;
  TYLO_REQUIRE(Mx && L, TYLO_ERR_INVALID_ARGUMENT, "%s: checkpoints Mx and L from the forward are required", who);
  TYLO_REQUIRE(!dEntropy || Entropy, TYLO_ERR_INVALID_ARGUMENT, "%s: dEntropy needs the forward's Entropy", who);
  LogprobArgs a = {};
  a.X = X; a.targets = targets; a.dX = dX; a.dLogp = dLogp; a.dEntropy = dEntropy; a.inEntropy = Entropy; a.inMx = Mx; a.inL = L;
  a.ldx = ldx; a.M = (int)M; a.temperature = temperature;
  TYLO_DISPATCH_DTYPE(dtype, T, return (logprob_bwd_dispatch<T>(who, a, N, (cudaStream_t)stream)));
  return TYLO_OK;
}

extern "C" int32_t tylo_b200_token_logprobs_fwd_bwd(float* Logp, float* Entropy, void* dX, const float* dLogp, const float* dEntropy,
                                                    const void* X, const int32_t* targets, int64_t M, int64_t N, int64_t ldx,
                                                    float temperature, int32_t dtype, tylo_stream_t stream) {
  const char* who = "token_logprobs_fwd_bwd";
  if (int32_t rc = check_vocab(who, X, M, N, ldx, temperature)) return rc;
  if (int32_t rc = check_vocab_grad(who, dX, X, M, N, ldx, dtype)) return rc;
  if (int32_t rc = check_logprob_weights(who, dLogp, dEntropy, targets)) return rc;
  TYLO_REQUIRE(!Logp || targets, TYLO_ERR_INVALID_ARGUMENT, "%s: Logp needs targets", who);
  TYLO_REQUIRE((!Logp || Logp != dLogp) && (!Entropy || Entropy != dEntropy), TYLO_ERR_INVALID_ARGUMENT,
               "%s: results and their weights must be different arrays", who);
  LogprobArgs a = {};
  a.X = X; a.targets = targets; a.Logp = Logp; a.Entropy = Entropy; a.dX = dX; a.dLogp = dLogp; a.dEntropy = dEntropy;
  a.ldx = ldx; a.M = (int)M; a.temperature = temperature;
  TYLO_DISPATCH_DTYPE(dtype, T, return (Entropy || dEntropy ? logprob_fwd_bwd_dispatch<T, true>(who, a, N, (cudaStream_t)stream)
                                                            : logprob_fwd_bwd_dispatch<T, false>(who, a, N, (cudaStream_t)stream)));
  return TYLO_OK;
}
