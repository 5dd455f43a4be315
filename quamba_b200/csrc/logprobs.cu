// Log probabilities of given tokens, entropy and likeliest alternatives from rows of logits, and their gradient (sm_100a).
//
// Forward: one pass over a row in 16-byte pieces.  With t = (x - m) log2 e for a reference m of the thread's own (raised when a
// value passes it by far), s = sum 2^t and w = sum t 2^t give
//   logprob = (x_target - m) - log2 s ln 2,   entropy = (log2 s - w / s) ln 2,
// in packed fp32 pairs: 3 to 4 issue slots and one MUFU result per value, against the 11 slots and 1.4 results that a 2-byte value
// leaves at the memory's speed.  Many rows take a CTA each; few rows a cluster of up to eight, whose parts are joined over
// distributed shared memory.
//
// Alternatives in the same pass.  The maxima of 64 groups of a CTA's threads over their first four pieces are ranked: the top_k-th of
// them is a bound that at least top_k values reach, so what is below it never counts again.  Values that reach it are listed
// (some tens), and the list is ranked at the end by (value, column).  A list that runs over (long plateaus of equal
// values, rows that rise to the end) sends the row's part to top_k searches for the largest key below the last.  A cluster's
// lists, each in order, are merged by bisection.
//
// Bound by the row's bytes, read once forward; read and written once backward: 8192 x 50280 fp16 128 us (6.5 TB/s), with the
// entropy 136; 4096 x 50288 bf16 with the entropy 75 us (5.5) and 149 us (5.5) back; 4096 x 50288 fp32 122 us (6.8) and 252 us.
// With alternatives by the phases between a CTA's barriers as well, of which three CTAs hide too little: 198 us for five of
// 8192 x 50280 fp16, 253 for twenty and the entropy.  Few rows are a chain of latencies: 8 x 50280 fp16 3.4 us, 6.8 with twenty
// alternatives and the entropy (first loads 1.0, bound 0.5, second reading 1.0, joining and ranking 1.2, cluster barrier 0.9, merging
// and answering 1.3).
#include <algorithm>
#include "common.cuh"

namespace qb {

int* device_status_ptr();

namespace {

constexpr int kStatusTarget = 502;       // keep in step with qb_read_device_status (lib.cu)
constexpr int kMaxCluster = 8;
constexpr int kGroups = 64;              // groups of threads whose first maxima are ranked (128: as many candidates, twice the time)
constexpr int kList = 2048;              // candidates listed per CTA
constexpr int kTop = QB_LOGPROBS_MAX_TOP;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFar = -1.0e4f;           // stands for everything below it where it is multiplied by a power that is zero there

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7fc00000); }

template <typename T> struct Wide { static constexpr int kN = 16 / sizeof(T); __align__(16) T v[kN]; };
__device__ __forceinline__ float val(float v) { return v; }
__device__ __forceinline__ float val(__half v) { return __half2float(v); }
__device__ __forceinline__ float val(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ void narrow2(float* p, float x, float y) { p[0] = x; p[1] = y; }
__device__ __forceinline__ void narrow2(__half* p, float x, float y) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x, y); }
__device__ __forceinline__ void narrow2(__nv_bfloat16* p, float x, float y) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x, y); }

template <typename T>
__device__ __forceinline__ Wide<T> load16(const T* p) {
  Wide<T> r;
  *reinterpret_cast<uint4*>(r.v) = *reinterpret_cast<const uint4*>(p);
  return r;
}
// the largest of a piece (a NaN beside numbers is passed over: it stays in the sums)
__device__ __forceinline__ float largest(const Wide<float>& r) { return fmaxf(fmaxf(r.v[0], r.v[1]), fmaxf(r.v[2], r.v[3])); }
__device__ __forceinline__ float largest(const Wide<__half>& r) {
  const __half2* h = reinterpret_cast<const __half2*>(r.v);
  const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return __half2float(__hmax(__low2half(m), __high2half(m)));
}
__device__ __forceinline__ float largest(const Wide<__nv_bfloat16>& r) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(r.v);
  const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return __bfloat162float(__hmax(__low2bfloat16(m), __high2bfloat16(m)));
}

struct Stats { float m, s, w; };         // m: the reference, -inf before the first number
// a headroom of e^kSlack costs s and w nothing: they are floats with exponents to spare
constexpr float kSlack = 16.0f;
__device__ __forceinline__ void raise(Stats& a, float m) {
  if (a.m != neg_inf()) {
    const float d = fmaxf((a.m - m) * kLog2e, kFar), f = fast_exp2(d);
    a.w = (a.w + a.s * d) * f;
    a.s *= f;
  }
  a.m = m;
}
__device__ __forceinline__ Stats join(Stats x, Stats y) {
  const float m = fmaxf(x.m, y.m);
  if (x.m != m) raise(x, m);               // a side without numbers (m = -inf) has s = w = 0, or a NaN
  if (y.m != m) raise(y, m);
  return Stats{m, x.s + y.s, x.w + y.w};
}
// a warp's, in every lane
__device__ __forceinline__ Stats join_warp(Stats x) {
  float m = x.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (x.m != m) raise(x, m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    x.s += __shfl_xor_sync(0xffffffffu, x.s, o);
    x.w += __shfl_xor_sync(0xffffffffu, x.w, o);
  }
  return x;
}
template <bool kEntropy>
__device__ __forceinline__ void add_one(Stats& a, float x) {
  if (x > a.m + kSlack) raise(a, x);
  const float t = (x - (a.m == neg_inf() ? 0.0f : a.m)) * kLog2e, e = fast_exp2(t);
  a.s += e;
  if (kEntropy) a.w = fmaf(e, fmaxf(t, kFar), a.w);
}
template <bool kEntropy, typename T>
__device__ __forceinline__ void add_piece(Stats& a, f2& s2, f2& w2, const Wide<T>& r, float top) {
  if (top > a.m + kSlack) {                // the pairs' sums go into the scalar ones first: they are relative to the old reference
    float x, y;
    unpack2(s2, x, y);
    a.s += x + y;
    unpack2(w2, x, y);
    a.w += x + y;
    s2 = w2 = 0ull;
    raise(a, top);
  }
  const float m = a.m == neg_inf() ? 0.0f : -a.m;
  const f2 mm = pack2(m, m), l2 = pack2(kLog2e, kLog2e);
#pragma unroll
  for (int k = 0; k < Wide<T>::kN; k += 2) {
    float x, y;
    const f2 t = mul2(add2(pack2(val(r.v[k]), val(r.v[k + 1])), mm), l2);   // not one fma: x log2 e may be out of range
    unpack2(t, x, y);
    const f2 e = pack2(fast_exp2(x), fast_exp2(y));          // NaN stays NaN
    s2 = add2(s2, e);
    if (kEntropy) w2 = fma2(e, pack2(fmaxf(x, kFar), fmaxf(y, kFar)), w2);
  }
}

// order-preserving key of (value, column): larger value first, then lower column; -0 counts as 0
__device__ __forceinline__ uint32_t rank_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float v, uint32_t col) { return ((uint64_t)rank_of(v) << 32) | (0xffffffffu - col); }
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ uint32_t column_of(uint64_t key) { return 0xffffffffu - (uint32_t)key; }
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// A part of a row: columns before the first 16-byte boundary, pieces, columns after the last.
template <typename T>
struct Part {
  const T* row;
  int begin, head, body, rest;             // columns [begin, begin + head), body pieces, rest columns in all besides the pieces
  __device__ __forceinline__ Part(const T* row_, int from, int to) : row(row_), begin(from) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + from) & 15;
    head = min(to - from, (int)(((16 - at) & 15) / sizeof(T)));
    body = (to - from - head) / Wide<T>::kN;
    rest = to - from - body * Wide<T>::kN;
  }
  __device__ __forceinline__ int piece(int i) const { return begin + head + i * Wide<T>::kN; }
  __device__ __forceinline__ int single(int i) const { return i < head ? begin + i : begin + i + body * Wide<T>::kN; }
};

// where row r begins (there are fewer than 2^31 rows, and a 64-bit division would hold a CTA's first load up)
__device__ __forceinline__ int64_t row_at(const qb_logprobs_args& a, uint32_t r, int64_t outer, int64_t inner) {
  const uint32_t n = (uint32_t)min(a.inner_rows, (int64_t)0x7fffffff), o = r / n;
  return o * outer + (r - o * n) * inner;
}

// the cluster's first CTA's copy of a shared variable (its own where there is no cluster)
template <typename V>
__device__ __forceinline__ V* cluster_first(V* mine) {
  uint64_t p;
  asm volatile("mapa.u64 %0, %1, 0;" : "=l"(p) : "l"(mine));
  return reinterpret_cast<V*>(p);
}

// Selecting the top_k of a part.
struct Select {
  uint32_t group[kGroups];
  uint64_t list[kList];
  uint64_t best[kMaxCluster * kTop];       // the winners of the cluster's CTAs, in the first one
  uint64_t warp_key[32];
  int count, found[kMaxCluster];
  float bound;
};

// A number that at least top_k of kGroups floats reach: the top_k-th largest, or for fp32 up to 2^-17 less, since the low bits
// of the order-preserving keys give way to the place, which makes them all different.
__device__ __forceinline__ uint32_t place_key(float v, int at) { return (rank_of(v) & ~(uint32_t)(kGroups - 1)) | (uint32_t)at; }
__device__ __forceinline__ void bound_of(const uint32_t* keys, int top_k, float* bound) {
  const int tid = (int)threadIdx.x;
  if (tid >= kGroups) return;
  const uint32_t mine = keys[tid];
  int above = 0;
#pragma unroll 4
  for (int j = 0; j < kGroups; j += 4) {
    const uint4 q = *reinterpret_cast<const uint4*>(keys + j);
    above += (q.x > mine) + (q.y > mine) + (q.z > mine) + (q.w > mine);
  }
  if (above == top_k - 1) *bound = value_of((uint64_t)max(mine & ~(uint32_t)(kGroups - 1), rank_of(neg_inf())) << 32);
}

// Without alternatives six CTAs of 256 threads an SM (40 registers): 8192 x 50280 fp16 131 us, where the five that 48 registers
// leave take 140; with the entropy 4096 x 50288 bf16 79 us against 89 at four.  Eight, or four rows of 16 bytes ahead made two,
// are no faster.
template <typename T, int kThreads, bool kEntropy, bool kAlt>
__global__ void __launch_bounds__(kThreads, kThreads == 64 ? 1 : kAlt ? 3 : 6) logprobs_kernel(const __grid_constant__ qb_logprobs_args a, int parts, int part_len, int* status) {
  constexpr int kWarps = kThreads / 32, kN = Wide<T>::kN, kAhead = 4;
  __shared__ Stats s_stats[kWarps], s_parts[kMaxCluster];
  __shared__ __align__(16) unsigned char s_select[kAlt ? sizeof(Select) : 16];
  Select& sel = *reinterpret_cast<Select*>(s_select);
  const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)(blockIdx.x % (uint32_t)parts);           // the cluster is `parts` neighbouring CTAs
  const uint32_t r = blockIdx.x / (uint32_t)parts;
  const T* const row = static_cast<const T*>(a.logits) + row_at(a, r, a.outer_stride, a.row_stride);
  const int from = rank * part_len, to = min(a.vocab, from + part_len);
  const Part<T> part(row, min(from, a.vocab), max(to, min(from, a.vocab)));

  const bool teller = tid == kThreads - 32 && rank == 0;   // not in the first warp: that one has alternatives to rank
  // asked for before the row and its value while the sums are joined: 128 us against 131 at 8192 x 50280 fp16, 3.4 against 3.7 at 8
  // rows; beside the alternatives' registers it costs more than it gives
  int64_t target = !kAlt && teller ? a.targets[r] : -1;
  if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  Stats st{neg_inf(), 0.0f, 0.0f};
  f2 s2 = 0ull, w2 = 0ull;
  float bound = neg_inf();
  const auto list_it = [&](float x, int c) {
    if (x >= bound && x > neg_inf()) {
      const int at = atomicAdd(&sel.count, 1);
      if (at < kList) sel.list[at] = key_of(x, (uint32_t)c);
    }
  };
  const auto look = [&](const Wide<T>& v, float top, int c) {
    if (!(top >= bound)) return;
    unsigned which = 0;
#pragma unroll
    for (int k = 0; k < kN; ++k) which |= val(v.v[k]) >= bound ? 1u << k : 0u;
    for (; which != 0; which &= which - 1) {             // one, as a rule; read again, which keeps this short code that rarely runs
      const int k = __ffs((int)which) - 1;
      list_it(val(row[c + k]), c + k);
    }
  };
  int i = tid;
  if (kAlt) {
    if (tid == 0) sel.count = 0;
    float over = neg_inf();                // a piece of nothing but NaN counts as -inf
    for (int j = tid; j < min(part.body, kAhead * kThreads); j += kThreads) over = fmaxf(over, largest(load16(row + part.piece(j))));
#pragma unroll
    for (int o = kThreads / kGroups / 2; o > 0; o /= 2) over = fmaxf(over, __shfl_xor_sync(0xffffffffu, over, o));
    if (tid % (kThreads / kGroups) == 0) sel.group[tid / (kThreads / kGroups)] = place_key(over, tid / (kThreads / kGroups));
    __syncthreads();
    bound_of(sel.group, a.top_k, &sel.bound);
    __syncthreads();
    bound = sel.bound;
  }
  for (; i + (kAhead - 1) * kThreads < part.body; i += kAhead * kThreads) {
    Wide<T> v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) v[j] = load16(row + part.piece(i + j * kThreads));
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const float top = largest(v[j]);
      add_piece<kEntropy>(st, s2, w2, v[j], top);
      if (kAlt) look(v[j], top, part.piece(i + j * kThreads));
    }
  }
  if (kAlt) {                              // the last pieces, fewer than kAhead a thread: one by one where the code is long
    for (; i < part.body; i += kThreads) {
      const Wide<T> v = load16(row + part.piece(i));
      const float top = largest(v);
      add_piece<kEntropy>(st, s2, w2, v, top);
      look(v, top, part.piece(i));
    }
  } else if (i < part.body) {
    Wide<T> v[kAhead - 1];
#pragma unroll
    for (int j = 0; j < kAhead - 1; ++j)
      if (i + j * kThreads < part.body) v[j] = load16(row + part.piece(i + j * kThreads));
#pragma unroll
    for (int j = 0; j < kAhead - 1; ++j) {
      if (i + j * kThreads >= part.body) break;
      add_piece<kEntropy>(st, s2, w2, v[j], largest(v[j]));
    }
  }
  {
    float x, y;
    unpack2(s2, x, y);
    st.s += x + y;
    unpack2(w2, x, y);
    st.w += x + y;
  }
  for (int j = tid; j < part.rest; j += kThreads) {
    const int c = part.single(j);
    const float x = val(row[c]);
    add_one<kEntropy>(st, x);
    if (kAlt) list_it(x, c);
  }
  float given = 0.0f;
  if (!kAlt && teller && target >= 0 && target < a.vocab) given = val(row[target]);
  st = join_warp(st);
  if (lane == 0) s_stats[warp] = st;
  __syncthreads();
  // The first CTA runs: its shared memory may be written.  (None of the cluster barriers is the .aligned form: that one wants whole
  // warps at a time, and lanes leave the loops over listed keys below one by one.)
  if (parts > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");

  int found = 0;
  if (kAlt) {                              // this part's best into the first CTA's sel.best, in order, zeros behind
    const int n = sel.count;
    uint64_t* const out = cluster_first(sel.best) + rank * kTop;
    found = min(n, a.top_k);
    if (n <= kList) {
      for (int j = tid; j < n; j += kThreads) {
        const uint64_t mine = sel.list[j];
        int above = 0;
        for (int k = 0; k < n; ++k) above += sel.list[k] > mine;
        if (above < a.top_k) out[above] = mine;
      }
    } else {
      uint64_t below = ~0ull;
      for (int k = 0; k < a.top_k; ++k) {
        uint64_t best = 0;
        const auto see = [&](float x, int c) {
          const uint64_t key = key_of(x, (uint32_t)c);
          if (x > neg_inf() && key < below && key > best) best = key;
        };
        for (int j = tid; j < part.body; j += kThreads) {
          const Wide<T> v = load16(row + part.piece(j));
#pragma unroll
          for (int e = 0; e < kN; ++e) see(val(v.v[e]), part.piece(j) + e);
        }
        for (int j = tid; j < part.rest; j += kThreads) see(val(row[part.single(j)]), part.single(j));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max64(best, (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)best, o));
        if (lane == 0) sel.warp_key[warp] = best;
        __syncthreads();
        for (int j = 0; j < kWarps; ++j) best = max64(best, sel.warp_key[j]);
        if (tid == 0) out[k] = best;
        below = best;
        __syncthreads();
      }
      found = a.top_k;                     // more than kList columns: there are as many
    }
    if (tid >= found && tid < kTop) out[tid] = 0;
    if (tid == 0) cluster_first(sel.found)[rank] = found;
  }
  if (parts > 1) {
    if (warp == 0) {
      st = join_warp(lane < kWarps ? s_stats[lane] : Stats{neg_inf(), 0.0f, 0.0f});
      if (lane == 0) cluster_first(s_parts)[rank] = st;
    }
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    if (rank != 0) return;
    st = join_warp(lane < parts ? s_parts[lane] : Stats{neg_inf(), 0.0f, 0.0f});
  } else {
    if (kAlt) __syncthreads();
    st = join_warp(lane < kWarps ? s_stats[lane] : Stats{neg_inf(), 0.0f, 0.0f});
  }
  const bool empty = st.m == neg_inf() && st.s == 0.0f;
  const float logs = log2f(st.s);
  const auto logprob = [&](float x) { return empty ? neg_inf() : fmaf(-logs, kLn2, x - st.m); };
  if (teller) {
    if (kAlt) target = a.targets[r];
    const bool inside = target >= 0 && target < a.vocab;
    if (kAlt && inside) given = val(row[target]);
    float lp = 0.0f;
    if (target != a.ignore_index) {
      lp = inside ? logprob(given) : quiet_nan();
      if (!inside) atomicCAS(status, 0, kStatusTarget);
    }
    a.logprobs[r] = lp;
    if (kEntropy) a.entropy[r] = empty ? 0.0f : (logs - st.w / st.s) * kLn2;
    if (a.lse != nullptr) a.lse[r] = empty ? neg_inf() : fmaf(logs, kLn2, st.m);
  }
  if (kAlt) {
    const auto answer = [&](int at, uint64_t key) {
      a.top_ids[(int64_t)r * a.top_k + at] = column_of(key);
      a.top_logprobs[(int64_t)r * a.top_k + at] = logprob(value_of(key));
    };
    int n = found;
    if (parts == 1) {
      if (tid < found) answer(tid, sel.best[tid]);
    } else {
      n = 0;
      for (int j = 0; j < parts; ++j) n += sel.found[j];
      // a key's place: how many of each part's keys are above it, by bisection in all parts at once
      for (int j = tid; j < parts * a.top_k; j += kThreads) {
        const uint64_t mine = sel.best[j % parts * kTop + j / parts];
        const uint64_t* at[kMaxCluster];   // the first key not known to be above
        int place = 0;
#pragma unroll
        for (int q = 0; q < kMaxCluster; ++q) at[q] = sel.best + min(q, parts - 1) * kTop;
#pragma unroll
        for (int step = kTop / 2; step > 0; step /= 2)
#pragma unroll
          for (int q = 0; q < kMaxCluster; ++q) at[q] += at[q][step - 1] > mine ? step : 0;
#pragma unroll
        for (int q = 0; q < kMaxCluster; ++q) place += q < parts ? (int)(at[q] - (sel.best + q * kTop)) + (*at[q] > mine) : 0;
        if (mine != 0 && place < a.top_k) answer(place, mine);
      }
    }
    // fewer numbers above -inf than asked for: the lowest of the other columns (-inf, or NaN in a row without a distribution)
    if (tid == 0)
      for (int c = 0; c < a.vocab && n < a.top_k; ++c) {
        const float x = val(row[c]);
        if (x > neg_inf()) continue;
        a.top_ids[(int64_t)r * a.top_k + n] = c;
        a.top_logprobs[(int64_t)r * a.top_k + n] = logprob(x);
        ++n;
      }
  }
}

// d_logits = g ([i == target] - p_i) - h p_i (log p_i + H); pieces of a row, kPieces per thread.  4096 x 50288 bf16 with the
// entropy's gradient: 151 us with five CTAs an SM, 161 with six (spills), 166 with four; fp32 255 us with six, 275 with five.
constexpr int kBwdThreads = 256, kPieces = 4;
template <typename T, bool kEntropy>
__global__ void __launch_bounds__(kBwdThreads, sizeof(T) == 2 ? 5 : 6) logprobs_bwd_kernel(const __grid_constant__ qb_logprobs_args a, int parts) {
  constexpr int kN = Wide<T>::kN;
  const uint32_t r = blockIdx.x / (uint32_t)parts;
  const int part = (int)(blockIdx.x % (uint32_t)parts);
  const T* row = static_cast<const T*>(a.logits) + row_at(a, r, a.outer_stride, a.row_stride);
  T* out = static_cast<T*>(a.d_logits) + row_at(a, r, a.d_outer_stride, a.d_row_stride);
  const int64_t t = a.targets[r];
  const bool kept = t != a.ignore_index && t >= 0 && t < a.vocab;
  const int target = kept ? (int)t : -1;
  const float g = kept && a.d_logprobs != nullptr ? a.d_logprobs[r] : 0.0f;
  const float h = kEntropy ? a.d_entropy[r] : 0.0f, H = kEntropy ? a.entropy[r] : 0.0f;
  const float lse = a.lse[r];
  const bool empty = lse == neg_inf();
  const float base = fmaf(h, H, g);                    // d = -p (g + h (log p + H))
  const f2 mm = pack2(-lse, -lse), l2 = pack2(kLog2e, kLog2e), hh = pack2(-h, -h), bb = pack2(-base, -base);
  auto two = [&](float x, float y) {
    const f2 lp = add2(pack2(x, y), mm);
    float u, v;
    unpack2(mul2(lp, l2), u, v);
    const f2 p = pack2(fast_exp2(u), fast_exp2(v));
    if (!kEntropy) return mul2(p, bb);
    unpack2(lp, u, v);
    return mul2(p, fma2(hh, pack2(fmaxf(u, kFar), fmaxf(v, kFar)), bb));
  };
  const uintptr_t ai = reinterpret_cast<uintptr_t>(row) & 15, ao = reinterpret_cast<uintptr_t>(out) & 15;
  const int head = ai == ao ? min(a.vocab, (int)((16 - ai) & 15) / (int)sizeof(T)) : a.vocab;   // not alike: one by one
  const int body = (a.vocab - head) / kN;
  // a CTA's share of the pieces: all that its threads take at once, or (fp32, 255 us against 268) as many as the others
  constexpr int kStep = kBwdThreads * kPieces;
  const int share = sizeof(T) == 2 ? kStep : (body / parts / kBwdThreads + 1) * kBwdThreads;
  const int from = part * share, to = min(body, from + share);
  for (int i0 = from; i0 < to; i0 += kStep) {
    Wide<T> v[kPieces];
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int i = i0 + k * kBwdThreads + (int)threadIdx.x;
      if (i < to) v[k] = load16(row + head + i * kN);
    }
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int i = i0 + k * kBwdThreads + (int)threadIdx.x, c = head + i * kN;
      if (i >= to) break;
      float d[kN];
#pragma unroll
      for (int j = 0; j < kN; j += 2) unpack2(two(val(v[k].v[j]), val(v[k].v[j + 1])), d[j], d[j + 1]);
      if (empty || (unsigned)(target - c) < (unsigned)kN)
#pragma unroll
        for (int j = 0; j < kN; ++j) d[j] = empty ? 0.0f : d[j] + (c + j == target ? g : 0.0f);
      Wide<T> o;
#pragma unroll
      for (int j = 0; j < kN; j += 2) narrow2(o.v + j, d[j], d[j + 1]);
      *reinterpret_cast<uint4*>(out + c) = *reinterpret_cast<const uint4*>(o.v);
    }
  }
  const int rest = a.vocab - body * kN;
  for (int i = part * kBwdThreads + (int)threadIdx.x; i < rest; i += parts * kBwdThreads) {
    const int c = i < head ? i : i + body * kN;
    float d, twin;
    unpack2(two(val(row[c]), 0.0f), d, twin);
    out[c] = narrow<T>(empty ? 0.0f : d + (c == target ? g : 0.0f));
  }
}

int check_logprobs(const qb_logprobs_args* a, const char* who) {
  QB_REQUIRE(a != nullptr, QB_ERR_INVALID_ARG, "%s: null pointer", who);
  QB_REQUIRE(a->rows >= 0 && a->vocab > 0 && (a->rows == 0 || a->inner_rows > 0), QB_ERR_INVALID_ARG, "%s: bad shape", who);
  QB_REQUIRE(a->vocab <= 1 << 30, QB_ERR_TOO_LARGE, "%s: more than 2^30 columns", who);        // a part more still fits an int
  QB_REQUIRE(a->dtype >= 0 && a->dtype <= 2, QB_ERR_INVALID_ARG, "%s: unsupported type", who);
  QB_REQUIRE(a->rows == 0 || (a->logits != nullptr && a->targets != nullptr), QB_ERR_INVALID_ARG, "%s: null pointer", who);
  QB_REQUIRE(aligned(a->logits, a->dtype == 0 ? 4 : 2), QB_ERR_INVALID_ARG, "%s: logits are not aligned to their type", who);
  return QB_OK;
}

template <typename T, int kThreads, bool kEntropy, bool kAlt>
int launch_logprobs(const qb_logprobs_args& a, int* status, cudaStream_t st) {
  // CTAs of a row: as many in all as are resident at once, with a piece per thread at least
  constexpr int kResident = kThreads == 64 ? 32 : kAlt ? 2 : 6;
  int64_t parts = 1;
  while (parts < kMaxCluster && a.rows * parts * 2 <= (int64_t)sm_count() * kResident && a.vocab / (parts * 2) >= kThreads * Wide<T>::kN) parts *= 2;
  const int64_t unit = 128 / (int64_t)sizeof(T), part_len = ceil_div(ceil_div(a.vocab, parts), unit) * unit;
  QB_REQUIRE(a.rows * parts < (1ll << 31), QB_ERR_TOO_LARGE, "logprobs_fwd: too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  (void)cudaLaunchKernelEx(&cfg, logprobs_kernel<T, kThreads, kEntropy, kAlt>, a, (int)parts, (int)part_len, status);
  QB_LAUNCH_OK("logprobs_kernel");
  return QB_OK;
}

template <typename T, int kThreads, int kAltThreads>
int launch_for(const qb_logprobs_args& a, int* status, cudaStream_t st) {
  if (a.top_k > 0) return a.entropy ? launch_logprobs<T, kAltThreads, true, true>(a, status, st) : launch_logprobs<T, kAltThreads, false, true>(a, status, st);
  return a.entropy ? launch_logprobs<T, kThreads, true, false>(a, status, st) : launch_logprobs<T, kThreads, false, false>(a, status, st);
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
    cudaStream_t st = (cudaStream_t)stream;
    // short rows take two warps: a CTA's set-up and reduction then weigh less
    return (int64_t)a->vocab * (int64_t)sizeof(T) < 16384 ? launch_for<T, 64, 64>(*a, status, st) : launch_for<T, 256, 512>(*a, status, st);
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
    if (a->d_entropy != nullptr) logprobs_bwd_kernel<T, true><<<(unsigned)(a->rows * parts), kBwdThreads, 0, (cudaStream_t)stream>>>(*a, (int)parts);
    else logprobs_bwd_kernel<T, false><<<(unsigned)(a->rows * parts), kBwdThreads, 0, (cudaStream_t)stream>>>(*a, (int)parts);
    QB_LAUNCH_OK("logprobs_bwd_kernel");
    return QB_OK;
  });
}
