// Log probabilities of given tokens, entropy and likeliest alternatives from rows of logits, and their gradient (sm_100a).
//
// One pass over a row with a running maximum m and, relative to it, s = sum exp(x - m) and w = sum exp(x - m) (x - m):
//   logprob = (x_target - m) - log s, entropy = log s - w / s.
// Bound by the row's bytes: read once forward; read and written once backward.
#include <algorithm>
#include "common.cuh"

namespace qb {

int* device_status_ptr();

namespace {

constexpr int kStatusTarget = 502;       // keep in step with qb_read_device_status (lib.cu)
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1.0e4f;           // stands for everything below it where it is multiplied by an exponential that is zero there

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

template <typename T> struct Wide { static constexpr int kN = 16 / sizeof(T); T v[kN]; };
__device__ __forceinline__ float val(float v) { return v; }
__device__ __forceinline__ float val(__half v) { return __half2float(v); }
__device__ __forceinline__ float val(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T>
__device__ __forceinline__ Wide<T> load16(const T* p) {
  Wide<T> r;
  *reinterpret_cast<uint4*>(r.v) = *reinterpret_cast<const uint4*>(p);
  return r;
}

struct Stats { float m, s, w; };
// m may be below the largest value by up to kSlack without harm: s and w are floats with exponents to spare
constexpr float kSlack = 16.0f;
__device__ __forceinline__ void raise(Stats& a, float m) {
  if (a.m != neg_inf()) {
    const float d = fmaxf(a.m - m, kFar), f = __expf(d);
    a.w = (a.w + a.s * d) * f;
    a.s *= f;
  }
  a.m = m;
}
template <int kN>
__device__ __forceinline__ void add(Stats& a, const float (&x)[kN]) {
  float top = x[0];
#pragma unroll
  for (int k = 1; k < kN; ++k) top = fmaxf(top, x[k]);
  if (top > a.m + kSlack) raise(a, top);              // always when a.m is still -inf and top is not
  const float m = a.m == neg_inf() ? 0.0f : a.m;
#pragma unroll
  for (int k = 0; k < kN; ++k) {
    const float d = x[k] - m, e = fast_exp2(d * kLog2e);   // NaN stays NaN
    a.s += e;
    a.w = fmaf(e, fmaxf(d, kFar), a.w);
  }
}
__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
  // by the larger maximum; an empty side (m = -inf) may still hold a NaN in s
  const float m = fmaxf(a.m, b.m);
  if (m == neg_inf()) return Stats{m, a.s + b.s, a.w + b.w};
  Stats x = a, y = b;
  if (x.m != m) { if (x.m == neg_inf()) x = Stats{m, a.s, a.w}; else raise(x, m); }
  if (y.m != m) { if (y.m == neg_inf()) y = Stats{m, b.s, b.w}; else raise(y, m); }
  return Stats{m, x.s + y.s, x.w + y.w};
}

// order-preserving key of (value, column): larger value first, then lower column; -0 counts as 0
__device__ __forceinline__ uint64_t key_of(float v, uint32_t col) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return ((uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32) | (0xffffffffu - col);
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ uint32_t column_of(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

// calls f(values, first column) over a row in 16-byte pieces, and over what lies before and after them one by one
template <typename T, typename F>
__device__ __forceinline__ void walk_row(const T* row, int vocab, int thread, int threads, F f) {
  constexpr int kN = Wide<T>::kN;
  const int head = min(vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
  const int body = (vocab - head) / kN;
  for (int i = thread; i < body; i += threads) {
    const Wide<T> r = load16(row + head + i * kN);
    float x[kN];
#pragma unroll
    for (int k = 0; k < kN; ++k) x[k] = val(r.v[k]);
    f(x, head + i * kN);
  }
  const int rest = vocab - body * kN;
  for (int i = thread; i < rest; i += threads) {
    const int c = i < head ? i : i + body * kN;
    const float x[1] = {val(row[c])};
    f(x, c);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const __grid_constant__ qb_logprobs_args a, int* status) {
  __shared__ Stats s_stats[kWarps];
  __shared__ uint64_t s_key[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* row = static_cast<const T*>(a.logits) + r / a.inner_rows * a.outer_stride + r % a.inner_rows * a.row_stride;
    Stats st{neg_inf(), 0.0f, 0.0f};
    walk_row(row, a.vocab, (int)threadIdx.x, kThreads, [&](const auto& x, int) { add(st, x); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      st = join(st, Stats{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.w, o)});
    if (lane == 0) s_stats[warp] = st;
    __syncthreads();
    st = s_stats[0];
    for (int i = 1; i < kWarps; ++i) st = join(st, s_stats[i]);
    const bool empty = st.m == neg_inf() && st.s == 0.0f;
    const float logs = logf(st.s);
    if (threadIdx.x == 0) {
      const int64_t t = a.targets[r];
      float lp = 0.0f;
      if (t != a.ignore_index) {
        if (t >= 0 && t < a.vocab) {
          lp = empty ? neg_inf() : (val(row[t]) - st.m) - logs;
        } else {
          lp = __int_as_float(0x7fc00000);
          atomicCAS(status, 0, kStatusTarget);
        }
      }
      a.logprobs[r] = lp;
      if (a.entropy != nullptr) a.entropy[r] = empty ? 0.0f : logs - st.w / st.s;
      if (a.lse != nullptr) a.lse[r] = empty ? neg_inf() : st.m + logs;
    }
    uint64_t below = ~0ull;
    for (int k = 0; k < a.top_k; ++k) {
      uint64_t best = 0;
      walk_row(row, a.vocab, (int)threadIdx.x, kThreads, [&](const auto& x, int c) {
#pragma unroll
        for (int j = 0; j < (int)(sizeof(x) / sizeof(float)); ++j) {
          const uint64_t key = key_of(x[j], (uint32_t)(c + j));
          if (key < below && key > best) best = key;
        }
      });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)best, o));
      if (lane == 0) s_key[warp] = best;
      __syncthreads();
      for (int i = 0; i < kWarps; ++i) best = max(best, s_key[i]);
      if (threadIdx.x == 0) {
        a.top_ids[r * a.top_k + k] = column_of(best);
        a.top_logprobs[r * a.top_k + k] = empty ? neg_inf() : (value_of(best) - st.m) - logs;
      }
      below = best;
      __syncthreads();
    }
    __syncthreads();
  }
}

// d_logits = g ([i == target] - p_i) - h p_i (log p_i + H); pieces of a row, kPieces vectors per thread
constexpr int kBwdThreads = 256, kPieces = 4;
template <typename T>
__global__ void __launch_bounds__(kBwdThreads) logprobs_bwd_kernel(const __grid_constant__ qb_logprobs_args a, int parts) {
  constexpr int kN = Wide<T>::kN;
  const int64_t r = blockIdx.x / parts;
  const int part = (int)(blockIdx.x % parts);
  const T* row = static_cast<const T*>(a.logits) + r / a.inner_rows * a.outer_stride + r % a.inner_rows * a.row_stride;
  T* out = static_cast<T*>(a.d_logits) + r / a.inner_rows * a.d_outer_stride + r % a.inner_rows * a.d_row_stride;
  const int64_t t = a.targets[r];
  const bool kept = t != a.ignore_index && t >= 0 && t < a.vocab;
  const float g = kept && a.d_logprobs != nullptr ? a.d_logprobs[r] : 0.0f;
  const float h = a.d_entropy != nullptr ? a.d_entropy[r] : 0.0f, H = a.d_entropy != nullptr ? a.entropy[r] : 0.0f;
  const float lse = a.lse[r];
  const bool empty = lse == neg_inf();
  const float base = fmaf(h, H, g);                    // d = -p (g + h (log p + H))
  auto one = [&](float x, int c) {
    const float lp = x - lse, p = fast_exp2(lp * kLog2e);
    float d = -p * fmaf(h, fmaxf(lp, kFar), base);
    if (c == t && kept) d += g;
    return empty ? 0.0f : d;
  };
  const uintptr_t ai = reinterpret_cast<uintptr_t>(row) & 15, ao = reinterpret_cast<uintptr_t>(out) & 15;
  const int head = ai == ao ? min(a.vocab, (int)((16 - ai) & 15) / (int)sizeof(T)) : a.vocab;   // not alike: one by one
  const int body = (a.vocab - head) / kN;
  constexpr int kStep = kBwdThreads * kPieces;
  for (int i0 = part * kStep; i0 < body; i0 += parts * kStep) {
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int i = i0 + k * kBwdThreads + (int)threadIdx.x;
      if (i < body) {
        const int c = head + i * kN;
        const Wide<T> v = load16(row + c);
        Wide<T> o;
#pragma unroll
        for (int j = 0; j < kN; ++j) o.v[j] = narrow<T>(one(val(v.v[j]), c + j));
        *reinterpret_cast<uint4*>(out + c) = *reinterpret_cast<const uint4*>(o.v);
      }
    }
  }
  const int rest = a.vocab - body * kN;
  for (int i = part * kBwdThreads + (int)threadIdx.x; i < rest; i += parts * kBwdThreads) {
    const int c = i < head ? i : i + body * kN;
    out[c] = narrow<T>(one(val(row[c]), c));
  }
}

int check_logprobs(const qb_logprobs_args* a, const char* who) {
  QB_REQUIRE(a != nullptr, QB_ERR_INVALID_ARG, "%s: null pointer", who);
  QB_REQUIRE(a->rows >= 0 && a->vocab > 0 && (a->rows == 0 || a->inner_rows > 0), QB_ERR_INVALID_ARG, "%s: bad shape", who);
  QB_REQUIRE(a->dtype >= 0 && a->dtype <= 2, QB_ERR_INVALID_ARG, "%s: unsupported type", who);
  QB_REQUIRE(a->rows == 0 || (a->logits != nullptr && a->targets != nullptr), QB_ERR_INVALID_ARG, "%s: null pointer", who);
  QB_REQUIRE(aligned(a->logits, a->dtype == 0 ? 4 : 2), QB_ERR_INVALID_ARG, "%s: logits are not aligned to their type", who);
  return QB_OK;
}

template <typename F>
int by_type(int dtype, F f) {
  return dtype == 0 ? f(float{}) : dtype == 1 ? f(__half{}) : f(__nv_bfloat16{});
}

}  // namespace
}  // namespace qb

using namespace qb;

extern "C" int qb_logprobs_fwd(const qb_logprobs_args* a, void* stream) {
  const int rc = check_logprobs(a, "logprobs_fwd");
  if (rc != QB_OK) return rc;
  QB_REQUIRE(a->top_k >= 0 && a->top_k <= QB_LOGPROBS_MAX_TOP && a->top_k <= a->vocab, QB_ERR_INVALID_ARG,
             "logprobs_fwd: top_k must be 0 to %d and at most the vocabulary, got %d", QB_LOGPROBS_MAX_TOP, a->top_k);
  if (a->rows == 0) return QB_OK;
  QB_REQUIRE(a->logprobs != nullptr && (a->top_k == 0 || (a->top_logprobs && a->top_ids)), QB_ERR_INVALID_ARG, "logprobs_fwd: null output");
  int* status = device_status_ptr();
  QB_REQUIRE(status != nullptr, QB_ERR_CUDA, "device status word unavailable");
  return by_type(a->dtype, [&](auto t) -> int {
    using T = decltype(t);
    logprobs_kernel<T><<<(unsigned)std::min<int64_t>(a->rows, 1 << 20), kThreads, 0, (cudaStream_t)stream>>>(*a, status);
    QB_LAUNCH_OK("logprobs_kernel");
    return QB_OK;
  });
}

extern "C" int qb_logprobs_bwd(const qb_logprobs_args* a, void* stream) {
  const int rc = check_logprobs(a, "logprobs_bwd");
  if (rc != QB_OK) return rc;
  if (a->rows == 0) return QB_OK;
  QB_REQUIRE(a->d_logits != nullptr && a->lse != nullptr && (a->d_entropy == nullptr || a->entropy != nullptr), QB_ERR_INVALID_ARG, "logprobs_bwd: null pointer");
  QB_REQUIRE(aligned(a->d_logits, a->dtype == 0 ? 4 : 2), QB_ERR_INVALID_ARG, "logprobs_bwd: d_logits is not aligned to its type");
  const int per = kBwdThreads * kPieces * (a->dtype == 0 ? 4 : 8);
  const int64_t parts = ceil_div(a->vocab, per);
  QB_REQUIRE(a->rows * parts < (1ll << 31), QB_ERR_TOO_LARGE, "logprobs_bwd: too many rows");
  return by_type(a->dtype, [&](auto t) -> int {
    using T = decltype(t);
    logprobs_bwd_kernel<T><<<(unsigned)(a->rows * parts), kBwdThreads, 0, (cudaStream_t)stream>>>(*a, (int)parts);
    QB_LAUNCH_OK("logprobs_bwd_kernel");
    return QB_OK;
  });
}
