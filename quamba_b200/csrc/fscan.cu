// Selective scan in floating point with gradients, channel-last (sm_100a): the Mamba1 recurrence of a float model.
//
//   delta = softplus(dt + bias), h_t[n] = exp(delta_t A[n]) h_{t-1}[n] + delta_t x_t B_t[n], y_t = (C_t . h_t + D x_t) silu(z_t)
//
// A warp owns a tile of channels of one sequence (or of a segment of it).  kQ lanes share kCh channels and hold kNp consecutive
// states of each: the states' sums over n are shuffles between two or four lanes, what a token's B and C cost is one or two
// 128-bit reads for all channels of a lane, and in the backward pass the sums over channels (dB, dC) are taken in the lane, then
// between the lanes, then over the CTA.  States and sums are float32 throughout, walked in packed pairs.
//
// Bound: dstate exponentials per (token, channel) on the MUFU pipe (16 results per clock and SM): 16 states cost 1 clock per
// (token, channel) and SM, while its bytes (8 at 16 bits) take 0.18 clocks of HBM time.
#include <algorithm>
#include <cstddef>
#include <type_traits>
#include "tc_common.cuh"

namespace qb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLift = 3.0e-8f;       // of the exponential unit: see make_up()
constexpr int kCkpt = 8;               // tokens between two kept states
constexpr int kBwdWarps = 4;

// kQ lanes share kCh channels; each holds kNp consecutive states of them.
template <int kNp_, int kCh_, int kQ_>
struct Geo {
  static constexpr int kNp = kNp_, kPairs = kNp / 2, kCh = kCh_, kQ = kQ_, kWc = 32 / kQ * kCh, kN = kQ * kNp;
  static constexpr int kLanesRow = kWc / 4;             // lanes that hold one token's channels, four each
  static constexpr int kRows = 32 / kLanesRow;          // tokens per warp-wide access
  static constexpr int kRec = 32 * kNp * kCh;           // states of a warp
  static constexpr int kSum = kRec + 32;                // a segment's summary: its states from zero, and the summed delta of its channels
  static constexpr int kGrad = kRec + 64;               // a warp's sums for dA | dD | d_bias
};

__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ f2 splat(float v) { return pack2(v, v); }
// max(v, 0) + log1p(e), e = exp(-|v|), for two values; log1p(e) = 2 artanh(s) with s = e / (2 + e) <= 1/3, by its series up to s^15
// (the next term is below 2^-29 of the sum).
__device__ __forceinline__ void softplus_series(float& a, float& b) {
  const f2 e = pack2(fast_exp2(-fabsf(a) * kLog2e), fast_exp2(-fabsf(b) * kLog2e));
  float x, y;
  unpack2(add2(e, splat(2.0f)), x, y);
  const f2 s = mul2(e, pack2(rcp_fast(x), rcp_fast(y))), w = mul2(s, s);
  f2 p = fma2(w, splat(1.0f / 15), splat(1.0f / 13));
  p = fma2(w, p, splat(1.0f / 11));
  p = fma2(w, p, splat(1.0f / 9));
  p = fma2(w, p, splat(1.0f / 7));
  p = fma2(w, p, splat(1.0f / 5));
  p = fma2(w, p, splat(1.0f / 3));
  p = fma2(w, p, splat(1.0f));
  unpack2(fma2(add2(s, s), p, pack2(fmaxf(a, 0.0f), fmaxf(b, 0.0f))), a, b);
}
__device__ __forceinline__ float sigmoid_fast(float v) { return rcp_fast(1.0f + fast_exp2(v * -kLog2e)); }
__device__ __forceinline__ f2 exp2_pair(f2 x) {
  float a, b;
  unpack2(x, a, b);
  return pack2(fast_exp2(a), fast_exp2(b));
}

// 2^x for two values with no systematic error where it would last: near zero, where a state lives long, by its series (|x| < 1/16: the
// term left out is below 2^-29), elsewhere from the exponential unit.
__device__ __forceinline__ f2 exp2_fine(f2 x) {
  f2 p = fma2(x, splat(9.6181291e-3f), splat(5.5504109e-2f));
  p = fma2(x, p, splat(0.24022651f));
  p = fma2(x, p, splat(kLn2));
  p = fma2(x, p, splat(1.0f));
  float a, b, u, v;
  unpack2(x, a, b);
  unpack2(p, u, v);
  return pack2(fabsf(a) < 0.0625f ? u : fast_exp2(a + kLift), fabsf(b) < 0.0625f ? v : fast_exp2(b + kLift));
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// four consecutive values in shared memory, 4 * sizeof(T) aligned
template <typename T>
__device__ __forceinline__ float4 quad(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    __align__(8) T v[4];
    *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(p);
    return make_float4(to_f(v[0]), to_f(v[1]), to_f(v[2]), to_f(v[3]));
  }
}
template <int kBytes>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "n"(kBytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory"); }

// `count` of four consecutive values to shared memory
template <bool kVec, typename T>
__device__ __forceinline__ void stage_quad(T* dst, const T* src, int count) {
  if constexpr (kVec) {
    if (count > 0) copy_async<4 * sizeof(T)>(dst, src);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < count) dst[k] = src[k];
  }
}

// four consecutive values to global memory, `count` of them where they do not lie together
template <typename T>
__device__ __forceinline__ void store_quad(T* dst, const float (&v)[4], int count, bool vec) {
  __align__(16) T r[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) r[k] = from_f<T>(v[k]);
  if (vec) {
    if (count > 0) {
      if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(r);
      else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(r);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < count) dst[k] = r[k];
  }
}

// consecutive floats of shared memory as pairs
template <int kPairs>
__device__ __forceinline__ void load_pairs(const float* p, f2 (&v)[kPairs]) {
#pragma unroll
  for (int i = 0; i < kPairs; i += 2) {
    const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(p + 2 * i);
    v[i] = w.x;
    v[i + 1] = w.y;
  }
}
template <int kCh>
__device__ __forceinline__ void load_channels(const float* p, float (&v)[kCh]) {
  if constexpr (kCh == 2) {
    const float2 w = *reinterpret_cast<const float2*>(p);
    v[0] = w.x; v[1] = w.y;
  } else {
    v[0] = *p;
  }
}

// v[c] summed over the kQ lanes of a group; the lane gets the total of the channel Place::own
template <int kCh, int kQ>
__device__ __forceinline__ float own_channel(const float (&v)[kCh], int q) {
  float a = v[0];
  int bit = kQ / 2;
  if constexpr (kCh == 2) {
    const bool hi = q & bit;
    a = (hi ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[1], bit);
    bit /= 2;
  }
#pragma unroll
  for (; bit > 0; bit /= 2) a += __shfl_xor_sync(0xffffffffu, a, bit);
  return a;
}

// A token's sums, over the lanes of one q, of kNp values each go to out: shuffles that halve the list at every step.  (Through shared
// memory they take fewer instructions but more time: 1.15 ms for 8 x 1024 tokens of 5120 channels of 16 states, 1.10 by shuffles.)
template <typename G>
__device__ __forceinline__ void group_sums(int lane, const f2 (&s)[G::kPairs], float* out) {
  float v[G::kNp];
#pragma unroll
  for (int p = 0; p < G::kPairs; ++p) unpack2(s[p], v[2 * p], v[2 * p + 1]);
  int at = 0, left = G::kNp;
#pragma unroll
  for (int bit = 16; bit >= G::kQ; bit >>= 1) {
    const bool up = lane & bit;
    if (left > 1) {
      left /= 2;
#pragma unroll
      for (int k = 0; k < left; ++k) v[k] = (up ? v[left + k] : v[k]) + __shfl_xor_sync(0xffffffffu, up ? v[k] : v[left + k], bit);
      at += up ? left : 0;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], bit);       // both hold the sum
    }
  }
#pragma unroll
  for (int k = 0; k < left; ++k) out[at + k] = v[k];
}

// a token's decays, and its step of the states
template <typename G>
__device__ __forceinline__ void decays(const float (&d)[G::kCh], const f2 (&A)[G::kCh][G::kPairs], f2 (&e)[G::kCh][G::kPairs]) {
  const f2 lift = pack2(kLift, kLift);                   // see make_up()
#pragma unroll
  for (int c = 0; c < G::kCh; ++c)
#pragma unroll
    for (int p = 0; p < G::kPairs; ++p) e[c][p] = fma2(pack2(d[c], d[c]), A[c][p], lift);
#pragma unroll
  for (int c = 0; c < G::kCh; ++c)
#pragma unroll
    for (int p = 0; p < G::kPairs; ++p) e[c][p] = exp2_pair(e[c][p]);
}
template <typename G>
__device__ __forceinline__ void advance(const f2 (&e)[G::kCh][G::kPairs], const float (&u)[G::kCh], const f2 (&b2)[G::kPairs], f2 (&h)[G::kCh][G::kPairs]) {
  f2 in[G::kCh][G::kPairs];
#pragma unroll
  for (int c = 0; c < G::kCh; ++c)
#pragma unroll
    for (int p = 0; p < G::kPairs; ++p) in[c][p] = mul2(b2[p], pack2(u[c], u[c]));
#pragma unroll
  for (int c = 0; c < G::kCh; ++c)
#pragma unroll
    for (int p = 0; p < G::kPairs; ++p) h[c][p] = fma2(e[c][p], h[c][p], in[c][p]);
}

// CTAs of the backward kernel on an SM: sixteen states a lane need 168 registers to stay out of local memory (four CTAs of 128: 12% slower)
template <typename G>
constexpr int kBwdBlocks = G::kNp * G::kCh == 16 ? 3 : 4;

// where a warp stands
template <typename G>
struct Place {
  int lane, q, cg;
  int b, seg, ch0, nch, group, tile;                     // the tile's first channel and how many exist
  int own;                                               // the channel (of the tile) whose sums this lane gets
  __device__ __forceinline__ Place(const qb_float_scan_args& a, int tpg, int b_, int seg_, int tile_, int lane_) {
    lane = lane_; q = lane % G::kQ; cg = lane / G::kQ;
    b = b_; seg = seg_; tile = tile_;
    const int per = a.dim / a.groups;
    group = tile / tpg;
    const int c0 = (tile % tpg) * G::kWc;
    ch0 = group * per + c0;
    nch = min(G::kWc, per - c0);
    own = cg * G::kCh + q * G::kCh / G::kQ;
  }
};

template <typename G>
__device__ __forceinline__ void load_A(const qb_float_scan_args& a, const Place<G>& w, f2 (&A)[G::kCh][G::kPairs]) {
#pragma unroll
  for (int c = 0; c < G::kCh; ++c)
#pragma unroll
    for (int p = 0; p < G::kPairs; ++p) {
      const int ch = w.cg * G::kCh + c, n = w.q * G::kNp + 2 * p;
      const float* row = a.A + (int64_t)(w.ch0 + ch) * a.dstate + n;
      const bool in = ch < w.nch;
      A[c][p] = pack2(in && n < a.dstate ? row[0] * kLog2e : 0.0f, in && n + 1 < a.dstate ? row[1] * kLog2e : 0.0f);
    }
}
// a (batch, dim, dstate) float32 tensor's part of this lane
template <typename G>
__device__ __forceinline__ void load_state(const float* s, const qb_float_scan_args& a, const Place<G>& w, f2 (&h)[G::kCh][G::kPairs]) {
#pragma unroll
  for (int c = 0; c < G::kCh; ++c)
#pragma unroll
    for (int p = 0; p < G::kPairs; ++p) {
      const int ch = w.cg * G::kCh + c, n = w.q * G::kNp + 2 * p;
      h[c][p] = 0ull;
      if (s != nullptr && ch < w.nch) {
        const float* row = s + ((int64_t)w.b * a.dim + w.ch0 + ch) * a.dstate + n;
        h[c][p] = pack2(n < a.dstate ? row[0] : 0.0f, n + 1 < a.dstate ? row[1] : 0.0f);
      }
    }
}
template <typename G>
__device__ __forceinline__ void store_state(float* s, const qb_float_scan_args& a, const Place<G>& w, const f2 (&h)[G::kCh][G::kPairs]) {
#pragma unroll
  for (int c = 0; c < G::kCh; ++c)
#pragma unroll
    for (int p = 0; p < G::kPairs; ++p) {
      const int ch = w.cg * G::kCh + c, n = w.q * G::kNp + 2 * p;
      if (ch >= w.nch) continue;
      float x, y;
      unpack2(h[c][p], x, y);
      float* row = s + ((int64_t)w.b * a.dim + w.ch0 + ch) * a.dstate + n;
      if (n < a.dstate) row[0] = x;
      if (n + 1 < a.dstate) row[1] = y;
    }
}
// a warp's states one after another, 16 bytes per lane and access
template <typename G, typename P>
__device__ __forceinline__ void load_record(const P* rec, int lane, f2 (&h)[G::kCh][G::kPairs]) {
#pragma unroll
  for (int i = 0; i < G::kCh * G::kPairs; i += 2) {
    const ulonglong2 v = __ldcg(reinterpret_cast<const ulonglong2*>(rec) + (i / 2) * 32 + lane);   // see grid_dependency_wait()
    h[i / G::kPairs][i % G::kPairs] = v.x;
    h[i / G::kPairs][i % G::kPairs + 1] = v.y;
  }
}
template <typename G, typename P>
__device__ __forceinline__ void store_record(P* rec, int lane, const f2 (&h)[G::kCh][G::kPairs]) {
#pragma unroll
  for (int i = 0; i < G::kCh * G::kPairs; i += 2)
    *(reinterpret_cast<ulonglong2*>(rec) + (i / 2) * 32 + lane) = make_ulonglong2(h[i / G::kPairs][i % G::kPairs], h[i / G::kPairs][i % G::kPairs + 1]);
}
// kept states lie as (batch, chunk, dim, 4 kNp), whatever a warp's share of the channels is
template <typename G>
__device__ __forceinline__ int64_t kept_at(const qb_float_scan_args& a, const Place<G>& w, int chunk) {
  return (((int64_t)w.b * ((a.seqlen + kCkpt - 1) / kCkpt) + chunk) * a.dim + w.ch0 + w.cg * G::kCh) * G::kN + w.q * G::kNp;
}
template <typename G>
__device__ __forceinline__ void load_kept(const qb_float_scan_args& a, const Place<G>& w, int chunk, f2 (&h)[G::kCh][G::kPairs]) {
  const float* at = a.checkpoints + kept_at(a, w, chunk);
#pragma unroll
  for (int c = 0; c < G::kCh; ++c)
#pragma unroll
    for (int p = 0; p < G::kPairs; p += 2) {
      ulonglong2 v = make_ulonglong2(0ull, 0ull);
      if (w.cg * G::kCh + c < w.nch) v = *reinterpret_cast<const ulonglong2*>(at + c * G::kN + 2 * p);
      h[c][p] = v.x;
      h[c][p + 1] = v.y;
    }
}
template <typename G>
__device__ __forceinline__ void store_kept(const qb_float_scan_args& a, const Place<G>& w, int chunk, const f2 (&h)[G::kCh][G::kPairs]) {
  float* at = a.checkpoints + kept_at(a, w, chunk);
#pragma unroll
  for (int c = 0; c < G::kCh; ++c)
#pragma unroll
    for (int p = 0; p < G::kPairs; p += 2)
      if (w.cg * G::kCh + c < w.nch) *reinterpret_cast<ulonglong2*>(at + c * G::kN + 2 * p) = make_ulonglong2(h[c][p], h[c][p + 1]);
}
// h <- what the summarised segment makes of it
template <typename G>
__device__ __forceinline__ void fold(const float* sum, const Place<G>& w, const f2 (&A)[G::kCh][G::kPairs], f2 (&h)[G::kCh][G::kPairs]) {
  f2 loc[G::kCh][G::kPairs];
  load_record<G>(sum, w.lane, loc);
#pragma unroll
  for (int c = 0; c < G::kCh; ++c) {
    const float d = __ldcg(sum + G::kRec + w.cg * G::kCh + c);
#pragma unroll
    for (int p = 0; p < G::kPairs; ++p) h[c][p] = fma2(exp2_pair(mul2(pack2(d, d), A[c][p])), h[c][p], loc[c][p]);
  }
}

// The exponential unit's results are low by 2.1e-8 of their value on average, one sign for all, which a state that lives for
// tens of tokens would lose for each of them; the exponent's fma adds that much (kLift).  For arguments in (-1/64, 0), where states
// live for hundreds of tokens, the mean error varies with the argument, by +-1.5e-8, and down to -3/64 it is a little larger:
// the difference is given back once for a tile of `tokens`, in its middle.  delta2 is the sum of two of the tile's deltas.  (The
// line below follows the mean error of 2^18 random arguments in each of 20 intervals.  Without all this the gradient of A is
// off by 2.8e-6, with it by less than 1e-6; a polynomial in place of the unit would cost 40% more instructions.)
template <typename G>
__device__ __forceinline__ void make_up(const float (&delta2)[G::kCh], float tokens, const f2 (&A)[G::kCh][G::kPairs], f2 (&h)[G::kCh][G::kPairs]) {
  const f2 rise = splat(3.4e-6f * tokens), rise0 = splat(-2.2e-8f * tokens);
  const float least = -1.51e-8f * tokens, most = 1.05e-8f * tokens, mid = 0.6e-8f * tokens;
#pragma unroll
  for (int c = 0; c < G::kCh; ++c) {
    const f2 half = splat(-0.5f * delta2[c]);
#pragma unroll
    for (int p = 0; p < G::kPairs; ++p) {
      const f2 arg = mul2(half, A[c][p]);                // A is negative
      float x, y, ux, uy;
      unpack2(arg, x, y);
      unpack2(fma2(arg, rise, rise0), ux, uy);
      ux = x < 1.0f / 64 ? fmaxf(fminf(ux, most), least) : x < 3.0f / 64 ? mid : 0.0f;
      uy = y < 1.0f / 64 ? fmaxf(fminf(uy, most), least) : y < 3.0f / 64 ? mid : 0.0f;
      h[c][p] = fma2(h[c][p], pack2(ux, uy), h[c][p]);
    }
  }
}

__device__ __forceinline__ int live_tokens(const qb_float_scan_args& a, int b) {
  return a.lengths != nullptr ? max(0, min(a.seqlen, a.lengths[b])) : a.seqlen;
}

// four tokens' or channels' delta before what is not there is left out
__device__ __forceinline__ void deltas(const float4& raw, const float (&bias)[4], int softplus, float (&d)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) d[k] = (k == 0 ? raw.x : k == 1 ? raw.y : k == 2 ? raw.z : raw.w) + bias[k];
  if (softplus) {
    softplus_series(d[0], d[1]);
    softplus_series(d[2], d[3]);
  }
}

struct Vec { int wide, bc; };           // whether four consecutive values can be moved together

// Raw rows of a tile of tokens, as they lie in memory.
template <typename T, typename G, int kT, int kWide>
struct Raw {
  T wide[kWide][kT][G::kWc];             // x, dt, z, dy
  T bc[2][kT][G::kN];
};
// stages tokens t0 .. min(t0 + kT, end) - 1
template <bool kVec, typename T, typename G, int kT, int kWide>
__device__ __forceinline__ void stage_wide(Raw<T, G, kT, kWide>& raw, const T* const (&src)[kWide], const int64_t (&stride)[kWide], int t0, int end, int nch, int lane) {
  const int row = lane / G::kLanesRow, c4 = (lane % G::kLanesRow) * 4;
#pragma unroll
  for (int k = 0; k < kWide; ++k) {
    if (src[k] == nullptr) continue;
    const T* at = src[k] + (int64_t)(t0 + row) * stride[k] + c4;
#pragma unroll
    for (int i = 0; i < (kT + G::kRows - 1) / G::kRows; ++i) {
      const int t = i * G::kRows + row;
      if (t < kT && t0 + t < end) stage_quad<kVec>(&raw.wide[k][t][c4], at + i * G::kRows * stride[k], nch - c4);
    }
  }
}
template <bool kVec, typename T, typename G, int kT, int kWide>
__device__ __forceinline__ void stage_bc(Raw<T, G, kT, kWide>& raw, const T* const (&bc)[2], const int64_t (&stride)[2], int t0, int end, int dstate, int lane) {
  constexpr int kQuads = G::kN / 4;
#pragma unroll
  for (int i = 0; i < 2 * kT * kQuads / 32; ++i) {
    const int e = i * 32 + lane, n4 = (e % kQuads) * 4, t = (e / kQuads) % kT, k = e / kQuads / kT;
    const T* from = k ? bc[1] : bc[0];
    if (t0 + t < end && from != nullptr) stage_quad<kVec>(&raw.bc[k][t][n4], from + (int64_t)(t0 + t) * (k ? stride[1] : stride[0]) + n4, dstate - n4);
  }
}
template <typename T, typename G, int kT, int kWide>
__device__ __forceinline__ void stage_tile(Raw<T, G, kT, kWide>& raw, const T* const (&src)[kWide], const int64_t (&stride)[kWide], const T* const (&bc)[2],
                                           const int64_t (&bc_stride)[2], int t0, int end, int nch, int dstate, Vec vec, int lane) {
  if (vec.wide) stage_wide<true, T, G, kT, kWide>(raw, src, stride, t0, end, nch, lane);
  else stage_wide<false, T, G, kT, kWide>(raw, src, stride, t0, end, nch, lane);
  if (vec.bc) stage_bc<true, T, G, kT, kWide>(raw, bc, bc_stride, t0, end, dstate, lane);
  else stage_bc<false, T, G, kT, kWide>(raw, bc, bc_stride, t0, end, dstate, lane);
}
// widens a tile's B and C, zero outside the sequence and past dstate
template <typename T, typename G, int kT, typename R>
__device__ __forceinline__ void widen_bc(const R& raw, float (&out)[2][kT][G::kN], int t0, int live, int dstate, int lane) {
  constexpr int kQuads = G::kN / 4;
#pragma unroll
  for (int i = 0; i < 2 * kT * kQuads / 32; ++i) {
    const int e = i * 32 + lane, n4 = (e % kQuads) * 4, t = (e / kQuads) % kT, k = e / kQuads / kT;
    float4 v = quad(&raw.bc[k][t][n4]);
    const bool in = t0 + t < live;
    v.x = in && n4 < dstate ? v.x : 0.0f;
    v.y = in && n4 + 1 < dstate ? v.y : 0.0f;
    v.z = in && n4 + 2 < dstate ? v.z : 0.0f;
    v.w = in && n4 + 3 < dstate ? v.w : 0.0f;
    *reinterpret_cast<float4*>(&out[k][t][n4]) = v;
  }
}
__device__ __forceinline__ float at(const float4& v, int k) { return k == 0 ? v.x : k == 1 ? v.y : k == 2 ? v.z : v.w; }


// ---- forward ----------------------------------------------------------------------------------------------------------------
template <typename T, typename G>
struct alignas(16) FwdSmem {
  static constexpr int kT = G::kRows <= 8 ? 8 : 16;   // tokens of a tile: one access per tensor at least
  Raw<T, G, kT, 3> raw[2];
  float delta[kT][G::kWc], u[kT][G::kWc];
  float bc[2][kT][G::kN];
};

// One warp: a tile of channels of one segment of one sequence.  kMode 0: outputs (from the folded summaries of the segments
// before); 1: the segment's summary; 2: the summary of the backward recurrence, from the segment's end to its start.
template <typename T, typename G, int kMode>
__global__ void __launch_bounds__(32, G::kRec == 512 ? 20 : 28)
float_scan_kernel(const __grid_constant__ qb_float_scan_args a, int tpg, int nseg, int seg_len, float* sums, Vec vec) {
  using S = FwdSmem<T, G>;
  constexpr int kT = S::kT, kNp = G::kNp;
  constexpr bool kOut = kMode == 0, kRev = kMode == 2;
  extern __shared__ __align__(16) unsigned char dyn[];
  S& s = *reinterpret_cast<S*>(dyn);
  const int tiles = tpg * a.groups;
  const int run = nseg - (kOut ? 0 : 1);                 // the last segment (the first, backwards) needs no summary
  const int seg_at = (int)(blockIdx.x / tiles) % run;
  const Place<G> w(a, tpg, (int)(blockIdx.x / tiles) / run, kRev ? seg_at + 1 : seg_at, (int)(blockIdx.x % tiles), (int)threadIdx.x);
  const int lane = w.lane;
  const int live = live_tokens(a, w.b);
  const int begin = w.seg * seg_len, end = min(a.seqlen, begin + seg_len);

  f2 A[G::kCh][G::kPairs], h[G::kCh][G::kPairs];
  load_A(a, w, A);
  load_state(kOut ? a.initial_state : nullptr, a, w, h);
  const T* const xp = static_cast<const T*>(kRev ? a.dy : a.x) + (int64_t)w.b * (kRev ? a.dy_sb : a.x_sb) + w.ch0;
  const T* const dp = static_cast<const T*>(a.dt) + (int64_t)w.b * a.dt_sb + w.ch0;
  const T* const zp = a.z != nullptr && kMode != 1 ? static_cast<const T*>(a.z) + (int64_t)w.b * a.z_sb + w.ch0 : nullptr;
  const T* const src[3] = {xp, dp, zp};
  const int64_t stride[3] = {kRev ? a.dy_sl : a.x_sl, a.dt_sl, a.z_sl};
  const T* const bc[2] = {kRev ? nullptr : static_cast<const T*>(a.Bm) + (int64_t)w.b * a.B_sb + (int64_t)w.group * a.B_sg,
                          kMode == 1 ? nullptr : static_cast<const T*>(a.Cm) + (int64_t)w.b * a.C_sb + (int64_t)w.group * a.C_sg};
  const int64_t bc_stride[2] = {a.B_sl, a.C_sl};

  const int row = lane / G::kLanesRow, c4 = (lane % G::kLanesRow) * 4;
  float bias[4], sum[4] = {};
#pragma unroll
  for (int k = 0; k < 4; ++k) bias[k] = a.dt_bias != nullptr && c4 + k < w.nch ? a.dt_bias[w.ch0 + c4 + k] : 0.0f;
  float Dv[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) Dv[k] = kOut && a.D != nullptr && c4 + k < w.nch ? a.D[w.ch0 + c4 + k] : 0.0f;
  const bool has_D = a.D != nullptr;
  T* const yp = kOut ? static_cast<T*>(a.y) + (int64_t)w.b * a.seqlen * a.dim + w.ch0 + c4 : nullptr;

  // The summaries' kernel lets the one that reads them in as it starts: everything up to the first tile's copy overlaps its end.
  if (!kOut) grid_dependency_launch();
  const int count = (int)((end - begin + kT - 1) / kT);
  auto tile_start = [&](int i) { return begin + (kRev ? count - 1 - i : i) * kT; };
  if (count > 0) stage_tile<T, G, kT, 3>(s.raw[0], src, stride, bc, bc_stride, tile_start(0), end, w.nch, a.dstate, vec, lane);
  copy_commit();
  if (kOut && nseg > 1) {
    grid_dependency_wait();
#pragma unroll 4
    for (int i = 0; i < w.seg; ++i) fold(sums + (((int64_t)w.b * nseg + i) * tiles + w.tile) * G::kSum, w, A, h);
  }
  for (int i = 0; i < count; ++i) {
    const int t0 = tile_start(i);
    auto& raw = s.raw[i & 1];
    if (i + 1 < count) stage_tile<T, G, kT, 3>(s.raw[(i + 1) & 1], src, stride, bc, bc_stride, tile_start(i + 1), end, w.nch, a.dstate, vec, lane);
    copy_commit();
    copy_wait<1>();
    __syncwarp();
    if (t0 < live) {
#pragma unroll
      for (int j = 0; j < kT / G::kRows; ++j) {
        const int t = j * G::kRows + row;
        const bool in = t0 + t < min(live, end);
        const float4 xv = quad(&raw.wide[0][t][c4]), dv = quad(&raw.wide[1][t][c4]);
        float4 zv;
        if (kRev && zp != nullptr) zv = quad(&raw.wide[2][t][c4]);
        float d[4], u[4];
        deltas(dv, bias, a.dt_softplus, d);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool on = in && c4 + k < w.nch;
          float g = at(xv, k) * (kRev ? 1.0f : d[k]);
          if (kRev && zp != nullptr) g *= at(zv, k) * sigmoid_fast(at(zv, k));
          d[k] = on ? d[k] : 0.0f;
          u[k] = on ? g : 0.0f;
          sum[k] += d[k];
        }
        *reinterpret_cast<float4*>(&s.delta[t][c4]) = make_float4(d[0], d[1], d[2], d[3]);
        *reinterpret_cast<float4*>(&s.u[t][c4]) = make_float4(u[0], u[1], u[2], u[3]);
      }
      widen_bc<T, G, kT>(raw, s.bc, t0, min(live, end), a.dstate, lane);
      __syncwarp();
#pragma unroll
      for (int half = 0; half < kT; half += kCkpt) {
        const int at0 = kRev ? kT - kCkpt - half : half, from = t0 + at0, lim = min(live, end);   // tokens from .. from + 7
        // the middle of 16 tokens (counted from the sequence's start, so that the way back meets the same states)
        if (kRev ? from % 16 == 0 && from + kCkpt < lim : from % 16 != 0 && from < lim) {
          float two[G::kCh], more[G::kCh];
          load_channels<G::kCh>(&s.delta[at0 + 1][w.cg * G::kCh], two);
          load_channels<G::kCh>(&s.delta[at0 + 5][w.cg * G::kCh], more);
#pragma unroll
          for (int c = 0; c < G::kCh; ++c) two[c] += more[c];
          make_up<G>(two, (float)min(16, lim - from / 16 * 16), A, h);
        }
        if (kOut && a.checkpoints != nullptr && from < lim && from > 0) store_kept(a, w, from / kCkpt, h);
#pragma unroll 1
        for (int j0 = half; j0 < half + kCkpt; j0 += 4) {
        float own[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = kRev ? kT - 1 - j0 - j : j0 + j;
          float d[G::kCh], u[G::kCh], y[G::kCh];
          f2 in2[G::kPairs], c2[G::kPairs], e[G::kCh][G::kPairs];
          load_channels<G::kCh>(&s.delta[t][w.cg * G::kCh], d);
          decays<G>(d, A, e);
          load_channels<G::kCh>(&s.u[t][w.cg * G::kCh], u);
          load_pairs<G::kPairs>(&s.bc[kRev ? 1 : 0][t][w.q * kNp], in2);
          if (kOut) load_pairs<G::kPairs>(&s.bc[1][t][w.q * kNp], c2);
          if (kRev) {
#pragma unroll
            for (int c = 0; c < G::kCh; ++c)
#pragma unroll
              for (int p = 0; p < G::kPairs; ++p) h[c][p] = mul2(e[c][p], fma2(in2[p], pack2(u[c], u[c]), h[c][p]));
          } else {
            f2 acc[G::kCh];
            advance<G>(e, u, in2, h);
#pragma unroll
            for (int p = 0; p < G::kPairs; ++p)
#pragma unroll
              for (int c = 0; c < G::kCh; ++c)
                if (kOut) acc[c] = p == 0 ? mul2(h[c][0], c2[0]) : fma2(h[c][p], c2[p], acc[c]);
#pragma unroll
            for (int c = 0; c < G::kCh; ++c) {
              float lo, hi;
              if (kOut) unpack2(acc[c], lo, hi), y[c] = lo + hi;
            }
          }
          if (kOut) own[j] = own_channel<G::kCh, G::kQ>(y, w.q);
        }
        if (kOut) {                                        // C . h takes the place of delta x, which these tokens no longer need
          __syncwarp();
          if (w.q % (G::kQ / G::kCh) == 0)
#pragma unroll
            for (int j = 0; j < 4; ++j) s.u[j0 + j][w.own] = own[j];
        }
        }
      }
      if (kOut) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < kT / G::kRows; ++j) {
          const int t = j * G::kRows + row;
          const float4 yv = quad(&s.u[t][c4]), xv = quad(&raw.wide[0][t][c4]);
          float4 zv;
          if (zp != nullptr) zv = quad(&raw.wide[2][t][c4]);
          float y[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = at(yv, k);
          if (has_D)
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = fmaf(Dv[k], at(xv, k), y[k]);
          if (zp != nullptr)
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] *= at(zv, k) * sigmoid_fast(at(zv, k));
          if (t0 + t >= live)
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = 0.0f;
          if (t0 + t < end) store_quad(yp + (int64_t)(t0 + t) * a.dim, y, w.nch - c4, vec.wide);
        }
      }
    } else if (kOut) {
      const float zero[4] = {};
#pragma unroll
      for (int j = 0; j < kT / G::kRows; ++j) {
        const int t = t0 + j * G::kRows + row;
        if (t < end) store_quad(yp + (int64_t)t * a.dim, zero, w.nch - c4, vec.wide);
      }
    }
    __syncwarp();
  }
  if (kOut) {
    if (a.final_state != nullptr && w.seg == nseg - 1) store_state(a.final_state, a, w, h);
  } else {
    float* rec = sums + (((int64_t)w.b * nseg + w.seg) * tiles + w.tile) * G::kSum;
    store_record<G>(rec, lane, h);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int o = G::kLanesRow; o < 32; o <<= 1) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
      if (row == 0) rec[G::kRec + c4 + k] = sum[k];
    }
  }
}

// ---- backward ---------------------------------------------------------------------------------------------------------------
// With g_t = dy_t silu(z_t) and dh_t = C_t g_t + a_{t+1} dh_{t+1}:
//   dC_t = sum_d g_t h_t, dB_t = sum_d dh_t delta_t x_t, dx_t = delta_t sum_n dh_t B_t + D g_t,
//   ddelta_t = x_t sum_n dh_t B_t + sum_n A (dh_t a_t h_{t-1}), dA = sum_t delta_t (dh_t a_t h_{t-1}).
// A warp walks its segment's chunks of eight tokens from the last to the first: forward once more from the state kept at the
// chunk's start, then back.  The eight states of the way forward (128 floats a lane) wait in tensor memory, which nothing else here uses: a warp
// reaches 32 of its lanes, one access moves a lane's 16 states, and 128 columns a CTA let four CTAs share an SM.  Kept in
// registers they cost all occupancy, in shared memory 4 KB of traffic per token and warp.
template <typename T, typename G>
struct alignas(16) BwdWarpSmem {            // one behind the other for the CTA's warps
  static constexpr int kT = kCkpt;
  static constexpr int kBuf = sizeof(T) == 2 ? 2 : 1;
  Raw<T, G, kT, 4> raw[kBuf];
  float delta[kT][G::kWc], u[kT][G::kWc], g[kT][G::kWc];
  float inner[kT][G::kWc], through[kT][G::kWc], into[kT][G::kWc];
  float bc[2][kT][G::kN];
  float part[kT][2][G::kN];
};

// a lane's 8 or 16 floats to and from its row of tensor memory
template <typename G>
__device__ __forceinline__ void tmem_keep(uint32_t at, const f2 (&h)[G::kCh][G::kPairs]) {
  uint32_t r[16];
#pragma unroll
  for (int i = 0; i < G::kCh * G::kPairs; ++i) {
    r[2 * i] = (uint32_t)h[i / G::kPairs][i % G::kPairs];
    r[2 * i + 1] = (uint32_t)(h[i / G::kPairs][i % G::kPairs] >> 32);
  }
  if constexpr (G::kRec == 512) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15])
                 : "memory");
  } else {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                 "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  }
}
template <typename G>
__device__ __forceinline__ void tmem_fetch(uint32_t at, uint32_t (&r)[16]) {
  if constexpr (G::kRec == 512) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at)
                 : "memory");
  } else {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(at)
                 : "memory");
  }
}
// waits for the fetch; its registers pass through here, so that nothing reads them before
template <typename G>
__device__ __forceinline__ void tmem_fetched(uint32_t (&r)[16], f2 (&h)[G::kCh][G::kPairs]) {
  tc::tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < G::kCh * G::kPairs; ++i) {
    asm volatile("" : "+r"(r[2 * i]), "+r"(r[2 * i + 1]));
    h[i / G::kPairs][i % G::kPairs] = (f2)r[2 * i] | ((f2)r[2 * i + 1] << 32);
  }
}
__device__ __forceinline__ void tmem_kept_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename T, typename G>
__global__ void __launch_bounds__(32 * kBwdWarps, kBwdBlocks<G>)
float_scan_bwd_kernel(const __grid_constant__ qb_float_scan_args a, int tpg, int nseg, int seg_len, const float* sums, float* part_bc, float* part_grad,
                      Vec vec) {
  using S = BwdWarpSmem<T, G>;
  static_assert(sizeof(S) % 16 == 0 && offsetof(S, delta) % 16 == 0 && offsetof(S, bc) % 16 == 0 && offsetof(S, part) % 16 == 0,
                "16-byte accesses");
  constexpr int kT = S::kT, kBuf = S::kBuf, kNp = G::kNp, kStates = G::kCh * kNp, kColumns = kT * kStates;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ uint32_t s_tmem;
  const int warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
  S& s = reinterpret_cast<S*>(dyn)[warp];
  if (warp == 0) {
    tc::tmem_alloc(&s_tmem, kColumns);
    tc::tmem_relinquish();
  }
  __syncthreads();
  const uint32_t tmem = s_tmem + ((uint32_t)warp << 21);        // the warp's 32 lanes of tensor memory
  const int cpg = (tpg + kBwdWarps - 1) / kBwdWarps, ctas = cpg * a.groups, tiles = tpg * a.groups;
  const int cta = (int)(blockIdx.x % ctas), rest = (int)(blockIdx.x / ctas);
  const int in_group = (cta % cpg) * kBwdWarps + warp;
  Place<G> w(a, tpg, rest / nseg, rest % nseg, (cta / cpg) * tpg + min(in_group, tpg - 1), lane);
  if (in_group >= tpg) w.nch = 0;                        // a warp past the group's last tile adds zeros to its CTA's sums
  const int live = live_tokens(a, w.b);
  const int begin = w.seg * seg_len, end = min(a.seqlen, begin + seg_len);

  f2 A[G::kCh][G::kPairs], carry[G::kCh][G::kPairs], dA[G::kCh][G::kPairs];
  load_A(a, w, A);
  load_state(a.d_final, a, w, carry);
  grid_dependency_launch();
  if (nseg > 1) grid_dependency_wait();
#pragma unroll 4
  for (int i = nseg - 1; i > w.seg; --i) fold(sums + (((int64_t)w.b * nseg + i) * tiles + w.tile) * G::kSum, w, A, carry);
#pragma unroll
  for (int c = 0; c < G::kCh; ++c)
#pragma unroll
    for (int p = 0; p < G::kPairs; ++p) dA[c][p] = 0ull;

  const int64_t at_out = (int64_t)w.b * a.seqlen * a.dim + w.ch0;
  const T* const src[4] = {static_cast<const T*>(a.x) + (int64_t)w.b * a.x_sb + w.ch0, static_cast<const T*>(a.dt) + (int64_t)w.b * a.dt_sb + w.ch0,
                           a.z != nullptr ? static_cast<const T*>(a.z) + (int64_t)w.b * a.z_sb + w.ch0 : nullptr,
                           static_cast<const T*>(a.dy) + (int64_t)w.b * a.dy_sb + w.ch0};
  const int64_t stride[4] = {a.x_sl, a.dt_sl, a.z_sl, a.dy_sl};
  const T* const bc[2] = {static_cast<const T*>(a.Bm) + (int64_t)w.b * a.B_sb + (int64_t)w.group * a.B_sg,
                          static_cast<const T*>(a.Cm) + (int64_t)w.b * a.C_sb + (int64_t)w.group * a.C_sg};
  const int64_t bc_stride[2] = {a.B_sl, a.C_sl};
  const bool has_z = a.z != nullptr, has_D = a.D != nullptr;
  const int row = lane / G::kLanesRow, c4 = (lane % G::kLanesRow) * 4;
  float bias[4], Dv[4], dD[4] = {}, dbias[4] = {};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    bias[k] = a.dt_bias != nullptr && c4 + k < w.nch ? a.dt_bias[w.ch0 + c4 + k] : 0.0f;
    Dv[k] = has_D && c4 + k < w.nch ? a.D[w.ch0 + c4 + k] : 0.0f;
  }
  T* const dxp = a.d_x != nullptr ? static_cast<T*>(a.d_x) + at_out + c4 : nullptr;
  T* const ddp = a.d_dt != nullptr ? static_cast<T*>(a.d_dt) + at_out + c4 : nullptr;
  T* const dzp = a.d_z != nullptr && has_z ? static_cast<T*>(a.d_z) + at_out + c4 : nullptr;
  float* const part = part_bc + ((int64_t)cta * a.batch + w.b) * a.seqlen * (2 * G::kN);

  const int first = begin / kT, last = (end + kT - 1) / kT - 1;
  // whole chunks past the sequence: zeros
  int chunk = last;
  for (; chunk >= first && chunk * kT >= live; --chunk) {
    const int lim = min(end, chunk * kT + kT);
    const float zero[4] = {};
    for (int t = chunk * kT + row; t < lim; t += G::kRows) {
      if (dxp != nullptr) store_quad(dxp + (int64_t)t * a.dim, zero, w.nch - c4, vec.wide);
      if (ddp != nullptr) store_quad(ddp + (int64_t)t * a.dim, zero, w.nch - c4, vec.wide);
      if (dzp != nullptr) store_quad(dzp + (int64_t)t * a.dim, zero, w.nch - c4, vec.wide);
    }
    for (int e = (int)threadIdx.x; e < (lim - chunk * kT) * 2 * G::kN; e += 32 * kBwdWarps) part[(int64_t)chunk * kT * 2 * G::kN + e] = 0.0f;
  }
  const int top = chunk;
  if (kBuf == 2) {
    if (top >= first) stage_tile<T, G, kT, 4>(s.raw[0], src, stride, bc, bc_stride, top * kT, end, w.nch, a.dstate, vec, lane);
    copy_commit();
  }
  for (; chunk >= first; --chunk) {
    const int t0 = chunk * kT, lim = min(live, end);
    auto& raw = s.raw[(top - chunk) % kBuf];
    if (kBuf == 2) {
      if (chunk > first)
        stage_tile<T, G, kT, 4>(s.raw[(top - chunk + 1) % kBuf], src, stride, bc, bc_stride, t0 - kT, end, w.nch, a.dstate, vec, lane);
      copy_commit();
      copy_wait<1>();
    } else {
      stage_tile<T, G, kT, 4>(raw, src, stride, bc, bc_stride, t0, end, w.nch, a.dstate, vec, lane);
      copy_commit();
      copy_wait<0>();
    }
    f2 h[G::kCh][G::kPairs];
    if (chunk == 0)
      load_state(a.initial_state, a, w, h);
    else
      load_kept(a, w, chunk, h);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < (kT + G::kRows - 1) / G::kRows; ++j) {
      const int t = j * G::kRows + row;
      if (t >= kT) break;
      const bool in = t0 + t < lim;
      const float4 xv = quad(&raw.wide[0][t][c4]), dv = quad(&raw.wide[1][t][c4]), yv = quad(&raw.wide[3][t][c4]);
      float4 zv;
      if (has_z) zv = quad(&raw.wide[2][t][c4]);
      float d[4], u[4], g[4];
      deltas(dv, bias, a.dt_softplus, d);
#pragma unroll
      for (int k = 0; k < 4; ++k) g[k] = at(yv, k);
      if (has_z)
#pragma unroll
        for (int k = 0; k < 4; ++k) g[k] *= at(zv, k) * sigmoid_fast(at(zv, k));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool on = in && c4 + k < w.nch;
        u[k] = on ? d[k] * at(xv, k) : 0.0f;
        d[k] = on ? d[k] : 0.0f;
        g[k] = on ? g[k] : 0.0f;
      }
      *reinterpret_cast<float4*>(&s.delta[t][c4]) = make_float4(d[0], d[1], d[2], d[3]);
      *reinterpret_cast<float4*>(&s.u[t][c4]) = make_float4(u[0], u[1], u[2], u[3]);
      *reinterpret_cast<float4*>(&s.g[t][c4]) = make_float4(g[0], g[1], g[2], g[3]);
    }
    widen_bc<T, G, kT>(raw, s.bc, t0, lim, a.dstate, lane);
    __syncwarp();
    // forward: C . h, and dC's sums over the warp's channels
#pragma unroll 2
    for (int t = 0; t < kT; ++t) {
      float d[G::kCh], u[G::kCh], g[G::kCh], y[G::kCh];
      f2 b2[G::kPairs], c2[G::kPairs], sC[G::kPairs], acc[G::kCh], e[G::kCh][G::kPairs];
      load_channels<G::kCh>(&s.delta[t][w.cg * G::kCh], d);
      decays<G>(d, A, e);
      load_channels<G::kCh>(&s.u[t][w.cg * G::kCh], u);
      load_channels<G::kCh>(&s.g[t][w.cg * G::kCh], g);
      load_pairs<G::kPairs>(&s.bc[0][t][w.q * kNp], b2);
      load_pairs<G::kPairs>(&s.bc[1][t][w.q * kNp], c2);
      tmem_keep<G>(tmem + t * kStates, h);
      advance<G>(e, u, b2, h);
#pragma unroll
      for (int p = 0; p < G::kPairs; ++p)
#pragma unroll
        for (int c = 0; c < G::kCh; ++c) {
          acc[c] = p == 0 ? mul2(h[c][0], c2[0]) : fma2(h[c][p], c2[p], acc[c]);
          sC[p] = c == 0 ? mul2(pack2(g[0], g[0]), h[0][p]) : fma2(pack2(g[c], g[c]), h[c][p], sC[p]);
        }
#pragma unroll
      for (int c = 0; c < G::kCh; ++c) {
        float lo, hi;
        unpack2(acc[c], lo, hi);
        y[c] = lo + hi;
      }
      const float own = own_channel<G::kCh, G::kQ>(y, w.q);
      if (w.q % (G::kQ / G::kCh) == 0) s.inner[t][w.own] = own;
      group_sums<G>(lane, sC, &s.part[t][1][w.q * kNp]);
    }
    tmem_kept_wait();
    // and back
#pragma unroll 2
    for (int t = kT - 1; t >= 0; --t) {
      float d[G::kCh], u[G::kCh], g[G::kCh], through[G::kCh], into[G::kCh];
      f2 b2[G::kPairs], c2[G::kPairs], sB[G::kPairs], e[G::kCh][G::kPairs], dh[G::kCh][G::kPairs], thr[G::kCh], q2[G::kCh];
      uint32_t kept[16];
      tmem_fetch<G>(tmem + t * kStates, kept);
      load_channels<G::kCh>(&s.delta[t][w.cg * G::kCh], d);
      decays<G>(d, A, e);
      load_channels<G::kCh>(&s.u[t][w.cg * G::kCh], u);
      load_channels<G::kCh>(&s.g[t][w.cg * G::kCh], g);
      load_pairs<G::kPairs>(&s.bc[0][t][w.q * kNp], b2);
      load_pairs<G::kPairs>(&s.bc[1][t][w.q * kNp], c2);
#pragma unroll
      for (int c = 0; c < G::kCh; ++c)
#pragma unroll
        for (int p = 0; p < G::kPairs; ++p) dh[c][p] = fma2(c2[p], pack2(g[c], g[c]), carry[c][p]);
#pragma unroll
      for (int c = 0; c < G::kCh; ++c)
#pragma unroll
        for (int p = 0; p < G::kPairs; ++p) carry[c][p] = mul2(dh[c][p], e[c][p]);
#pragma unroll
      for (int p = 0; p < G::kPairs; ++p)
#pragma unroll
        for (int c = 0; c < G::kCh; ++c) {
          sB[p] = c == 0 ? mul2(pack2(u[0], u[0]), dh[0][p]) : fma2(pack2(u[c], u[c]), dh[c][p], sB[p]);
          thr[c] = p == 0 ? mul2(dh[c][0], b2[0]) : fma2(dh[c][p], b2[p], thr[c]);
        }
      tmem_fetched<G>(kept, h);
#pragma unroll
      for (int p = 0; p < G::kPairs; ++p)
#pragma unroll
        for (int c = 0; c < G::kCh; ++c) {
          dh[c][p] = mul2(carry[c][p], h[c][p]);
          q2[c] = p == 0 ? mul2(dh[c][0], A[c][0]) : fma2(dh[c][p], A[c][p], q2[c]);
          dA[c][p] = fma2(dh[c][p], pack2(d[c], d[c]), dA[c][p]);
        }
#pragma unroll
      for (int c = 0; c < G::kCh; ++c) {
        float lo, hi;
        unpack2(thr[c], lo, hi);
        through[c] = lo + hi;
        unpack2(q2[c], lo, hi);
        into[c] = lo + hi;
      }
      group_sums<G>(lane, sB, &s.part[t][0][w.q * kNp]);
      const float own_through = own_channel<G::kCh, G::kQ>(through, w.q), own_into = own_channel<G::kCh, G::kQ>(into, w.q);
      if (w.q % (G::kQ / G::kCh) == 0) {
        s.through[t][w.own] = own_through;
        s.into[t][w.own] = own_into;
      }
    }
    if (chunk % 2 == 1) {                                // the middle of a tile of the forward pass
      float two[G::kCh], more[G::kCh];
      load_channels<G::kCh>(&s.delta[1][w.cg * G::kCh], two);
      load_channels<G::kCh>(&s.delta[5][w.cg * G::kCh], more);
#pragma unroll
      for (int c = 0; c < G::kCh; ++c) two[c] += more[c];
      make_up<G>(two, (float)min(2 * kT, lim - t0 + kT), A, carry);
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < (kT + G::kRows - 1) / G::kRows; ++j) {
      const int t = j * G::kRows + row;
      if (t >= kT) break;
      const bool in = t0 + t < lim;
      const float4 th = quad(&s.through[t][c4]), it = quad(&s.into[t][c4]), al = quad(&s.inner[t][c4]), dl = quad(&s.delta[t][c4]), gv = quad(&s.g[t][c4]);
      const float4 xv = quad(&raw.wide[0][t][c4]), dv = quad(&raw.wide[1][t][c4]), yv = quad(&raw.wide[3][t][c4]);
      float4 zv;
      if (has_z) zv = quad(&raw.wide[2][t][c4]);
      float dx[4], dd[4], dz[4], x[4], slope[4] = {1.0f, 1.0f, 1.0f, 1.0f};
      bool on[4];
      if (a.dt_softplus)
#pragma unroll
        for (int k = 0; k < 4; ++k) slope[k] = sigmoid_fast(at(dv, k) + bias[k]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        on[k] = in && c4 + k < w.nch;
        x[k] = on[k] ? at(xv, k) : 0.0f;
        dx[k] = fmaf(Dv[k], at(gv, k), at(th, k) * at(dl, k));
        dd[k] = fmaf(at(th, k), x[k], at(it, k) * kLn2) * slope[k];
        dd[k] = on[k] ? dd[k] : 0.0f;
        dx[k] = on[k] ? dx[k] : 0.0f;
        dD[k] = fmaf(at(gv, k), x[k], dD[k]);
        dbias[k] += dd[k];
      }
      if (has_z)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float sig = sigmoid_fast(at(zv, k));
          const float full = fmaf(Dv[k], x[k], at(al, k));
          dz[k] = at(yv, k) * full * sig * fmaf(at(zv, k), 1.0f - sig, 1.0f);
          dz[k] = on[k] ? dz[k] : 0.0f;
        }
      if (t0 + t < end) {
        const int64_t at_t = (int64_t)(t0 + t) * a.dim;
        if (dxp != nullptr) store_quad(dxp + at_t, dx, w.nch - c4, vec.wide);
        if (ddp != nullptr) store_quad(ddp + at_t, dd, w.nch - c4, vec.wide);
        if (dzp != nullptr) store_quad(dzp + at_t, dz, w.nch - c4, vec.wide);
      }
    }
    // the CTA's channels together
    __syncthreads();
    const S* all = reinterpret_cast<const S*>(dyn);
    for (int i = (int)threadIdx.x; i < (min(end, t0 + kT) - t0) * 2 * G::kN; i += 32 * kBwdWarps) {
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < kBwdWarps; ++k) v += (&all[k].part[0][0][0])[i];
      part[(int64_t)t0 * 2 * G::kN + i] = v;
    }
    __syncthreads();
  }
  if (w.nch > 0) {
    float* rec = part_grad + (((int64_t)w.b * nseg + w.seg) * tiles + w.tile) * G::kGrad;
    store_record<G>(rec, lane, dA);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int o = G::kLanesRow; o < 32; o <<= 1) {
        dD[k] += __shfl_xor_sync(0xffffffffu, dD[k], o);
        dbias[k] += __shfl_xor_sync(0xffffffffu, dbias[k], o);
      }
      if (row == 0) {
        rec[G::kRec + c4 + k] = dD[k];
        rec[G::kRec + 32 + c4 + k] = dbias[k];
      }
    }
    if (a.d_initial != nullptr && w.seg == 0) store_state(a.d_initial, a, w, carry);
  }
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(s_tmem, kColumns);
}

// dB and dC: the CTAs' sums added up in their order
template <typename T>
__global__ void __launch_bounds__(256) float_scan_bc_kernel(const __grid_constant__ qb_float_scan_args a, const float* part, int cpg, int npad) {
  grid_dependency_launch();
  grid_dependency_wait();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;      // (b, t, group, B | C, n)
  const int n = (int)(i % npad), k = (int)(i / npad % 2), g = (int)(i / (2 * npad) % a.groups);
  const int64_t bt = i / ((int64_t)2 * npad * a.groups), tokens = (int64_t)a.batch * a.seqlen;
  if (bt >= tokens || n >= a.dstate) return;
  const float* p = part + ((int64_t)g * cpg * tokens + bt) * (2 * npad) + k * npad + n;
  float v = 0.0f;
  for (int c = 0; c < cpg; ++c) v += __ldcg(p + (int64_t)c * tokens * (2 * npad));
  T* out = static_cast<T*>(k ? a.d_C : a.d_B);
  if (out != nullptr) out[(bt * a.groups + g) * a.dstate + n] = from_f<T>(v);
}

// dA, dD, d_bias: summed over sequences and segments in their order
template <typename G>
__global__ void __launch_bounds__(G::kGrad) float_scan_param_kernel(const __grid_constant__ qb_float_scan_args a, const float* part, int tpg, int runs) {
  constexpr int kRec = G::kRec, kGrad = G::kGrad, kNp = G::kNp;
  grid_dependency_wait();
  const int tiles = tpg * a.groups, tile = (int)blockIdx.x, i = (int)threadIdx.x;
  const int per = a.dim / a.groups, c0 = (tile % tpg) * G::kWc, ch0 = tile / tpg * per + c0, nch = min(G::kWc, per - c0);
  const bool is_A = i < kRec;
  // a record's float4 k of lane l holds the values 4 k .. 4 k + 3 of that lane, value = channel of the lane * kNp + state
  const int l = i / 4 % 32, v = i / 128 * 4 + i % 4;
  const int ch = is_A ? l / G::kQ * G::kCh + v / kNp : (i - kRec) % 32, n = is_A ? l % G::kQ * kNp + v % kNp : 0;
  if (ch >= nch || (is_A && n >= a.dstate)) return;
  const float* p = part + (int64_t)tile * kGrad + i;
  float sum = 0.0f;
  for (int r = 0; r < runs; ++r) sum += __ldcg(p + (int64_t)r * tiles * kGrad);
  if (is_A) {
    if (a.d_A != nullptr) a.d_A[(int64_t)(ch0 + ch) * a.dstate + n] = sum;
  } else if (i < kRec + 32) {
    if (a.d_D != nullptr) a.d_D[ch0 + ch] = sum;
  } else if (a.d_bias != nullptr) {
    a.d_bias[ch0 + ch] = sum;
  }
}

// ---- one token --------------------------------------------------------------------------------------------------------------
// Bound by the state, read and written once (8 bytes per state): 256 sequences of 5120 channels of 16 states 37 us (4.5 TB/s), 64 12 us;
// what is left are the latencies of a turn (eight warps more an SM or the next turn's states in L2 already change nothing).  kLanes lanes
// of a channel hold four states each and walk `rows` sequences, kAhead at a time: all loads first, none of them widened or asked for under
// a condition, which would wait for each in turn (52 us).  Two at a time and eight CTAs an SM: four and six 39 us.  What a (sequence,
// channel) costs besides its states -- loads, softplus, gate, output -- a lane does for its own share of the kAhead sequences only, and passes delta and delta x round.
constexpr int kAhead = 2, kUpdateBlocks = 8;
// Four values as whole registers, where they lie together.
template <typename T> struct Packed { using type = uint2; };
template <> struct Packed<float> { using type = float4; };
template <bool kVec, typename T>
__device__ __forceinline__ typename Packed<T>::type load_packed(const T* p, int count) {
  using R = typename Packed<T>::type;
  if constexpr (kVec) {
    return *reinterpret_cast<const R*>(p);
  } else {
    __align__(16) T v[4] = {};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < count) v[k] = p[k];
    return *reinterpret_cast<const R*>(v);
  }
}
template <typename T>
__device__ __forceinline__ void widen(const typename Packed<T>::type& r, f2& lo, f2& hi) {
  __align__(16) T v[4];
  *reinterpret_cast<typename Packed<T>::type*>(v) = r;
  lo = pack2(to_f(v[0]), to_f(v[1]));
  hi = pack2(to_f(v[2]), to_f(v[3]));
}
template <typename T, int kLanes, bool kVec>
__global__ void __launch_bounds__(128, kUpdateBlocks) float_update_kernel(const __grid_constant__ qb_float_update_args a, int rows) {
  constexpr int kOwners = kLanes < kAhead ? kLanes : kAhead, kOwn = kAhead / kOwners;
  const int i = (int)blockIdx.x * 128 + (int)threadIdx.x;
  const int sub = i % kLanes, n0 = min(sub * 4, kVec ? a.dstate - 4 : 64), count = a.dstate - sub * 4, d = min(i / kLanes, a.dim - 1), g = d / (a.dim / a.groups);   // the last lanes repeat the last channel
  const bool mine = i / kLanes == d;
  f2 A[2];
  {
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = k < count ? a.A[(int64_t)d * a.dstate + n0 + k] * kLog2e : 0.0f;
    A[0] = pack2(v[0], v[1]);
    A[1] = pack2(v[2], v[3]);
  }
  const float bias = a.dt_bias != nullptr ? a.dt_bias[d] : 0.0f, Dv = a.D != nullptr ? a.D[d] : 0.0f;
  const int b0 = (int)blockIdx.y * rows, b1 = min(a.batch, b0 + rows), own0 = min(sub, kOwners - 1) * kOwn;
  const float* st = a.state + (int64_t)d * a.state_sd + n0;
  float* so = a.state_out + (int64_t)d * a.state_out_sd + n0;
  const T* Bp = static_cast<const T*>(a.Bm) + (int64_t)g * a.B_sg + n0;
  const T* Cp = static_cast<const T*>(a.Cm) + (int64_t)g * a.C_sg + n0;
  for (int c0 = b0; c0 < b1; c0 += kAhead) {
    float4 h[kAhead];
    typename Packed<T>::type B[kAhead], C[kAhead];
    T xr[kOwn], dr[kOwn], zr[kOwn];
    float x[kOwn], dl[kOwn], z[kOwn], u[kOwn], own_y[kOwn];
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const int64_t b = min(c0 + own0 + k, b1 - 1);      // past the last: the last again
      xr[k] = static_cast<const T*>(a.x)[b * a.x_sb + d];
      dr[k] = static_cast<const T*>(a.dt)[b * a.dt_sb + d];
      zr[k] = a.z != nullptr ? static_cast<const T*>(a.z)[b * a.z_sb + d] : from_f<T>(0.0f);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t b = min(c0 + k, b1 - 1);
      h[k] = load_packed<kVec>(st + b * a.state_sb, count);
      B[k] = load_packed<kVec>(Bp + b * a.B_sb, count);
      C[k] = load_packed<kVec>(Cp + b * a.C_sb, count);
    }
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      x[k] = to_f(xr[k]);
      z[k] = to_f(zr[k]);
      dl[k] = to_f(dr[k]) + bias;
      float twin = dl[k];
      if (a.dt_softplus) softplus_series(dl[k], twin);
      u[k] = dl[k] * x[k];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      // one decay a call: what is systematic in it would add up over calls (see make_up())
      const f2 dd = splat(__shfl_sync(0xffffffffu, dl[k % kOwn], k / kOwn, kLanes)), uu = splat(__shfl_sync(0xffffffffu, u[k % kOwn], k / kOwn, kLanes));
      f2 in0, in1, out0, out1;
      widen<T>(B[k], in0, in1);
      widen<T>(C[k], out0, out1);
      const f2 h0 = fma2(exp2_fine(mul2(dd, A[0])), pack2(h[k].x, h[k].y), mul2(uu, in0));
      const f2 h1 = fma2(exp2_fine(mul2(dd, A[1])), pack2(h[k].z, h[k].w), mul2(uu, in1));
      float y, y1;
      unpack2(fma2(h1, out1, mul2(h0, out0)), y, y1);
      y = count > 0 ? y + y1 : 0.0f;
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
      if (k / kOwn == min(sub, kOwners - 1)) own_y[k % kOwn] = y;
      if (mine && c0 + k < b1) {
        float4 r;
        unpack2(h0, r.x, r.y);
        unpack2(h1, r.z, r.w);
        float* to = so + (c0 + k) * a.state_out_sb;
        if (kVec) {
          if (count > 0) *reinterpret_cast<float4*>(to) = r;
        } else {
          if (0 < count) to[0] = r.x;
          if (1 < count) to[1] = r.y;
          if (2 < count) to[2] = r.z;
          if (3 < count) to[3] = r.w;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const int b = c0 + own0 + k;
      float y = own_y[k];
      if (a.D != nullptr) y = fmaf(Dv, x[k], y);
      if (a.z != nullptr) y *= z[k] * sigmoid_fast(z[k]);
      if (mine && b < b1 && sub < kOwners) static_cast<T*>(a.y)[(int64_t)b * a.dim + d] = from_f<T>(y);
    }
  }
}

// ---- host -------------------------------------------------------------------------------------------------------------------
// How the work is dealt out.
struct Plan {
  int np, ch, q;                           // Geo
  int tpg, tiles, nseg, seg_len;
  int rec() const { return 32 * np * ch; }
  int wide() const { return np * q; }
};
constexpr int kMinSeg = 32;                // tokens of a segment, at least
constexpr int kMaxSegs = 32;               // a segment folds the summaries of all on its one side

Plan share_of(int batch, int dim, int groups, int np, int ch, int q) {
  Plan p{np, ch, q, 0, 0, 1, 0};
  p.tpg = (int)ceil_div(dim / groups, 32 / q * ch);
  p.tiles = p.tpg * groups;
  return p;
}
void cut(Plan& p, int seqlen, int64_t want) {
  const int64_t n = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, kMaxSegs), seqlen / kMinSeg));
  p.seg_len = (int)std::max<int64_t>(16, ceil_div(ceil_div(seqlen, n), 16) * 16);
  p.nseg = (int)std::max<int64_t>(1, ceil_div(seqlen, p.seg_len));
}
// Forward.  Eight states a lane: sixteen take fewer instructions but leave too few warps on an SM to hide each one's latencies
// (8 x 1024 tokens of 5120 channels: 367 us against 440).  More than 32 states: eight of two channels, as on the way back (2 x 1024 tokens of
// 5120 channels: 409 us, sixteen of one channel 511, eight of one 689).  Rows that put fewer than eight warps on an SM are cut into segments, which are
// walked twice (512 tokens of 1536 channels: 23 us, in one piece 68; 4 x 2048 of 5120, nine warps: 482, cut in four 532).  Pieces of 32
// tokens are the shortest (2 x 333 tokens of 1536 channels: 28 us, of 64 34, of 16 27, but 4 x 256 33, 38 and 36).  What fewer than six warps
// an SM are left of then takes four states a lane.
Plan plan_fwd(int batch, int seqlen, int dim, int groups, int dstate) {
  Plan p = dstate <= 16 ? share_of(batch, dim, groups, 8, 1, 2) : dstate <= 32 ? share_of(batch, dim, groups, 8, 1, 4) : share_of(batch, dim, groups, 8, 2, 8);
  const int64_t sms = sm_count();
  if (dstate <= 16 && (int64_t)batch * p.tiles < 8 * sms && (int64_t)batch * p.tiles * std::max(1, seqlen / kMinSeg) < 12 * sms)
    p = share_of(batch, dim, groups, 4, 1, 4);
  const int64_t warps = std::max<int64_t>(1, (int64_t)batch * p.tiles);
  cut(p, seqlen, warps >= 8 * sms ? 1 : ceil_div(32 * sms, warps));
  return p;
}
// Backward: sixteen states a lane, in as many segments as make the number of waves of resident CTAs (three an SM) times a segment's
// length smallest; pieces of fewer than 64 tokens only while all are in one wave (1024 tokens of 300 channels: 44 us, 60 with pieces of 64;
// 8 x 128 of 4096 in one piece 128, in three 148).  A segment's summary costs a quarter of its walk.  8 x 1024 tokens of 5120 channels:
// 1.07 ms, in one piece 1.54; 16384 of 2048 fp32: 0.93 ms in 27 segments, 1.05 in 24, 1.13 with eight states a lane.  Where even the most segments leave an SM fewer
// than eight warps, eight a lane (2 x 333 tokens of 1536 channels: 66 us against 72; 4 x 256, ten warps: 79 against 73).
// Up to 64 states lie on eight lanes of two channels (2 x 1024 tokens of 5120 channels: 1.13 ms; sixteen a lane of one channel, with twice
// the reads of B and C: 1.76).
Plan plan_bwd(int batch, int seqlen, int dim, int groups, int dstate) {
  const int64_t sms = sm_count();
  Plan p = dstate <= 16 ? share_of(batch, dim, groups, 8, 2, 2) : dstate <= 32 ? share_of(batch, dim, groups, 8, 2, 4) : share_of(batch, dim, groups, 8, 2, 8);
  if (dstate <= 32 && (int64_t)batch * p.tiles * std::min(kMaxSegs, std::max(1, seqlen / kMinSeg)) < 8 * sms) p = share_of(batch, dim, groups, 8, 1, p.q);
  const int64_t ctas = std::max<int64_t>(1, (int64_t)batch * groups * ceil_div(p.tpg, kBwdWarps)), slots = (p.ch == 2 ? 3 : 4) * sms;
  int64_t best = 1;
  double least = 0.0;
  for (int64_t n = 1; n <= std::min<int64_t>(kMaxSegs, std::max(1, seqlen / kMinSeg)); ++n) {
    if (seqlen / n < 2 * kMinSeg && n > 1 && ctas * n > slots) break;
    const double cost = (double)ceil_div(ctas * n, slots) / n * (1.0 + 0.25 * (n - 1) / n);
    if (n == 1 || cost < least) { least = cost; best = n; }
  }
  cut(p, seqlen, best);
  return p;
}
Plan plan_of(int batch, int seqlen, int dim, int groups, int dstate, bool backward) {
  return backward ? plan_bwd(batch, seqlen, dim, groups, dstate) : plan_fwd(batch, seqlen, dim, groups, dstate);
}
int64_t align256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t sums_bytes(const Plan& p, int64_t batch) { return p.nseg > 1 ? align256(batch * p.nseg * p.tiles * (p.rec() + 32) * (int64_t)sizeof(float)) : 0; }
int64_t part_bytes(const Plan& p, int64_t batch, int64_t seqlen, int groups) {
  return align256(ceil_div(p.tpg, kBwdWarps) * groups * batch * seqlen * 2 * p.wide() * (int64_t)sizeof(float));
}
int64_t grad_bytes(const Plan& p, int64_t batch) { return align256(batch * p.nseg * p.tiles * (p.rec() + 64) * (int64_t)sizeof(float)); }

bool sizes_ok(int64_t batch, int64_t seqlen, int64_t dim, int64_t groups, int64_t dstate) {
  return batch >= 0 && seqlen >= 0 && dim > 0 && groups > 0 && dim % groups == 0 && dstate >= 1 && dstate <= 64;
}
bool quads(const void* p, int64_t s1, int64_t s2, size_t size) { return p == nullptr || (aligned(p, 4 * size) && s1 % 4 == 0 && s2 % 4 == 0); }

int check_scan(const qb_float_scan_args* a, bool backward) {
  const char* who = backward ? "float_scan_bwd" : "float_scan_fwd";
  QB_REQUIRE(a != nullptr && a->x && a->dt && a->Bm && a->Cm && a->A, QB_ERR_INVALID_ARG, "%s: null pointer", who);
  QB_REQUIRE(a->dstate >= 1 && a->dstate <= 64, QB_ERR_INVALID_ARG, "%s: dstate must be 1 to 64, got %d", who, a->dstate);
  QB_REQUIRE(a->batch >= 0 && a->seqlen >= 0 && a->dim > 0 && a->groups > 0, QB_ERR_INVALID_ARG, "%s: bad shape", who);
  QB_REQUIRE(a->seqlen <= 1 << 30, QB_ERR_TOO_LARGE, "%s: more than 2^30 tokens in a sequence", who);   // a tile or segment more still fits an int
  QB_REQUIRE(a->dim % a->groups == 0, QB_ERR_INVALID_ARG, "%s: dim = %d is not divisible by groups = %d", who, a->dim, a->groups);
  QB_REQUIRE(a->dtype >= 0 && a->dtype <= 2, QB_ERR_INVALID_ARG, "%s: unsupported type", who);
  const Plan p = plan_of(a->batch, a->seqlen, a->dim, a->groups, a->dstate, backward);
  QB_REQUIRE((int64_t)a->batch * p.nseg * p.tiles < (1ll << 31), QB_ERR_TOO_LARGE, "%s: batch and dim are too large", who);
  return QB_OK;
}
Vec vec_of(const qb_float_scan_args& a, bool backward) {
  const size_t size = a.dtype == 0 ? 4 : 2;
  const bool wide = a.dim / a.groups % 4 == 0 && quads(a.x, a.x_sb, a.x_sl, size) && quads(a.dt, a.dt_sb, a.dt_sl, size) && quads(a.z, a.z_sb, a.z_sl, size) &&
                    (!backward || quads(a.dy, a.dy_sb, a.dy_sl, size));
  const bool bc = a.dstate % 4 == 0 && quads(a.Bm, a.B_sb, a.B_sl, size) && quads(a.Cm, a.C_sb, a.C_sl, size) && a.B_sg % 4 == 0 && a.C_sg % 4 == 0;
  return Vec{wide, bc};
}

template <typename T, typename G, int kMode>
int launch_scan(const qb_float_scan_args& a, const Plan& p, float* sums, Vec vec, cudaStream_t st) {
  const size_t smem = sizeof(FwdSmem<T, G>);
  static PerDeviceOnce attr;
  const int rc = attr.run([&]() -> int {
    QB_CUDA_OK(cudaFuncSetAttribute(float_scan_kernel<T, G, kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    return QB_OK;
  });
  if (rc != QB_OK) return rc;
  const int64_t grid = (int64_t)a.batch * (p.nseg - (kMode == 0 ? 0 : 1)) * p.tiles;
  if (kMode == 0 && p.nseg > 1) launch_dependent(float_scan_kernel<T, G, kMode>, dim3((unsigned)grid), dim3(32), smem, st, a, p.tpg, p.nseg, p.seg_len, sums, vec);
  else float_scan_kernel<T, G, kMode><<<(unsigned)grid, 32, smem, st>>>(a, p.tpg, p.nseg, p.seg_len, sums, vec);
  QB_LAUNCH_OK("float_scan_kernel");
  return QB_OK;
}

template <typename T, typename G>
int run_fwd(const qb_float_scan_args& a, const Plan& p, cudaStream_t st) {
  float* sums = static_cast<float*>(a.workspace);
  const Vec vec = vec_of(a, false);
  if (p.nseg > 1) {
    const int rc = launch_scan<T, G, 1>(a, p, sums, vec, st);
    if (rc != QB_OK) return rc;
  }
  return launch_scan<T, G, 0>(a, p, sums, vec, st);
}

template <typename T, typename G>
int run_bwd(const qb_float_scan_args& a, const Plan& p, cudaStream_t st) {
  unsigned char* ws = static_cast<unsigned char*>(a.workspace);
  float* sums = reinterpret_cast<float*>(ws);
  float* part = reinterpret_cast<float*>(ws + sums_bytes(p, a.batch));
  float* grad = reinterpret_cast<float*>(ws + sums_bytes(p, a.batch) + part_bytes(p, a.batch, a.seqlen, a.groups));
  const Vec vec = vec_of(a, true);
  if (p.nseg > 1 && a.batch > 0) {
    const int rc = launch_scan<T, G, 2>(a, p, sums, vec, st);
    if (rc != QB_OK) return rc;
  }
  const size_t smem = sizeof(BwdWarpSmem<T, G>) * kBwdWarps;
  static PerDeviceOnce attr;
  const int rc = attr.run([&]() -> int {
    QB_CUDA_OK(cudaFuncSetAttribute(float_scan_bwd_kernel<T, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    return QB_OK;
  });
  if (rc != QB_OK) return rc;
  const int cpg = (int)ceil_div(p.tpg, kBwdWarps);
  if (a.batch > 0) {
    const int64_t grid = (int64_t)a.batch * p.nseg * cpg * a.groups;
    if (p.nseg > 1) launch_dependent(float_scan_bwd_kernel<T, G>, dim3((unsigned)grid), dim3(32 * kBwdWarps), smem, st, a, p.tpg, p.nseg, p.seg_len, sums, part, grad, vec);
    else float_scan_bwd_kernel<T, G><<<(unsigned)grid, 32 * kBwdWarps, smem, st>>>(a, p.tpg, p.nseg, p.seg_len, sums, part, grad, vec);
    QB_LAUNCH_OK("float_scan_bwd_kernel");
  }
  const int64_t cells = (int64_t)a.batch * a.seqlen * a.groups * 2 * G::kN;
  if (cells > 0 && (a.d_B != nullptr || a.d_C != nullptr)) {
    launch_dependent(float_scan_bc_kernel<T>, dim3((unsigned)ceil_div(cells, 256)), dim3(256), 0, st, a, part, cpg, G::kN);
    QB_LAUNCH_OK("float_scan_bc_kernel");
  }
  if (a.d_A != nullptr || a.d_D != nullptr || a.d_bias != nullptr) {
    launch_dependent(float_scan_param_kernel<G>, dim3((unsigned)p.tiles), dim3(G::kGrad), 0, st, a, grad, p.tpg, a.batch * p.nseg);
    QB_LAUNCH_OK("float_scan_param_kernel");
  }
  return QB_OK;
}

template <typename F>
int by_type(int dtype, F f) {
  return dtype == 0 ? f(float{}) : dtype == 1 ? f(__half{}) : f(__nv_bfloat16{});
}
template <typename F>
int by_share_fwd(const Plan& p, F f) {
  if (p.np == 4) return f(Geo<4, 1, 4>{});
  return p.q == 2 ? f(Geo<8, 1, 2>{}) : p.q == 4 ? f(Geo<8, 1, 4>{}) : f(Geo<8, 2, 8>{});
}
template <typename F>
int by_share_bwd(const Plan& p, F f) {
  if (p.ch == 1) return p.q == 2 ? f(Geo<8, 1, 2>{}) : f(Geo<8, 1, 4>{});
  return p.q == 2 ? f(Geo<8, 2, 2>{}) : p.q == 4 ? f(Geo<8, 2, 4>{}) : f(Geo<8, 2, 8>{});
}

}  // namespace
}  // namespace qb

using namespace qb;

extern "C" int64_t qb_float_scan_checkpoint_bytes(int32_t batch, int32_t seqlen, int32_t dim, int32_t groups, int32_t dstate) {
  if (!sizes_ok(batch, seqlen, dim, groups, dstate)) return -1;
  return (int64_t)batch * ceil_div(seqlen, kCkpt) * dim * (dstate <= 16 ? 16 : dstate <= 32 ? 32 : 64) * (int64_t)sizeof(float);
}

extern "C" int64_t qb_float_scan_workspace_bytes(int32_t batch, int32_t seqlen, int32_t dim, int32_t groups, int32_t dstate, int32_t backward) {
  if (!sizes_ok(batch, seqlen, dim, groups, dstate)) return -1;
  const Plan p = plan_of(batch, seqlen, dim, groups, dstate, backward != 0);
  return sums_bytes(p, batch) + (backward ? part_bytes(p, batch, seqlen, groups) + grad_bytes(p, batch) : 0);
}

extern "C" int qb_float_scan_fwd(const qb_float_scan_args* a, void* stream) {
  const int rc = check_scan(a, false);
  if (rc != QB_OK) return rc;
  QB_REQUIRE(a->y != nullptr || (int64_t)a->batch * a->seqlen == 0, QB_ERR_INVALID_ARG, "float_scan_fwd: null output");
  if (a->batch == 0) return QB_OK;
  const Plan p = plan_of(a->batch, a->seqlen, a->dim, a->groups, a->dstate, false);
  const int64_t need = sums_bytes(p, a->batch);
  QB_REQUIRE(need == 0 || (a->workspace != nullptr && a->workspace_bytes >= need && aligned(a->workspace, 16)), QB_ERR_INVALID_ARG,
             "float_scan_fwd: the workspace must have %lld bytes, 16-byte aligned", (long long)need);
  QB_REQUIRE(aligned(a->checkpoints, 16), QB_ERR_INVALID_ARG, "float_scan_fwd: checkpoints must be 16-byte aligned");
  return by_type(a->dtype, [&](auto t) -> int {
    using T = decltype(t);
    cudaStream_t st = (cudaStream_t)stream;
    return by_share_fwd(p, [&](auto g) -> int { return run_fwd<T, decltype(g)>(*a, p, st); });
  });
}

extern "C" int qb_float_scan_bwd(const qb_float_scan_args* a, void* stream) {
  const int rc = check_scan(a, true);
  if (rc != QB_OK) return rc;
  QB_REQUIRE((a->dy != nullptr && a->checkpoints != nullptr) || (int64_t)a->batch * a->seqlen == 0, QB_ERR_INVALID_ARG, "float_scan_bwd: dy and checkpoints are needed");
  QB_REQUIRE(aligned(a->checkpoints, 16), QB_ERR_INVALID_ARG, "float_scan_bwd: checkpoints must be 16-byte aligned");
  const Plan p = plan_of(a->batch, a->seqlen, a->dim, a->groups, a->dstate, true);
  const int64_t need = sums_bytes(p, a->batch) + part_bytes(p, a->batch, a->seqlen, a->groups) + grad_bytes(p, a->batch);
  QB_REQUIRE(need == 0 || (a->workspace != nullptr && a->workspace_bytes >= need && aligned(a->workspace, 16)), QB_ERR_INVALID_ARG,
             "float_scan_bwd: the workspace must have %lld bytes, 16-byte aligned", (long long)need);
  return by_type(a->dtype, [&](auto t) -> int {
    using T = decltype(t);
    cudaStream_t st = (cudaStream_t)stream;
    return by_share_bwd(p, [&](auto g) -> int { return run_bwd<T, decltype(g)>(*a, p, st); });
  });
}

extern "C" int qb_float_scan_update(const qb_float_update_args* a, void* stream) {
  QB_REQUIRE(a != nullptr && a->state && a->state_out && a->x && a->dt && a->Bm && a->Cm && a->A && a->y, QB_ERR_INVALID_ARG, "float_scan_update: null pointer");
  QB_REQUIRE(sizes_ok(a->batch, 1, a->dim, a->groups, a->dstate), QB_ERR_INVALID_ARG,
             "float_scan_update: bad shape (dstate 1 to 64, dim divisible by groups)");
  QB_REQUIRE(a->dtype >= 0 && a->dtype <= 2, QB_ERR_INVALID_ARG, "float_scan_update: unsupported type");
  if (a->batch == 0) return QB_OK;
  const int lanes = a->dstate <= 4 ? 1 : a->dstate <= 8 ? 2 : a->dstate <= 16 ? 4 : a->dstate <= 32 ? 8 : 16;
  const int64_t across = ceil_div((int64_t)a->dim * lanes, 128);
  // sequences of a thread, in whole turns of kAhead: as many as make all CTAs resident at once
  const int64_t share = ceil_div(a->batch, std::min<int64_t>(a->batch, std::max<int64_t>(1, kUpdateBlocks * sm_count() / across)));
  const int64_t rows = share > 2 ? ceil_div(share, kAhead) * kAhead : share, down = ceil_div(a->batch, rows);
  QB_REQUIRE(across < (1ll << 24) && down < 65536, QB_ERR_TOO_LARGE, "float_scan_update: batch and dim are too large");
  const size_t size = a->dtype == 0 ? 4 : 2;
  const bool vec = a->dstate % 4 == 0 && aligned(a->state, 16) && aligned(a->state_out, 16) &&
                   (a->state_sb | a->state_sd | a->state_out_sb | a->state_out_sd) % 4 == 0 &&
                   aligned(a->Bm, 4 * size) && aligned(a->Cm, 4 * size) && (a->B_sb | a->B_sg | a->C_sb | a->C_sg) % 4 == 0;
  return by_type(a->dtype, [&](auto t) -> int {
    using T = decltype(t);
    cudaStream_t st = (cudaStream_t)stream;
    const dim3 g((unsigned)across, (unsigned)down);
    const auto go = [&](auto lanes_, auto vec_) {
      float_update_kernel<T, decltype(lanes_)::value, decltype(vec_)::value><<<g, 128, 0, st>>>(*a, (int)rows);
    };
    const auto pick = [&](auto vec_) {
      if (lanes == 1) go(std::integral_constant<int, 1>{}, vec_);
      else if (lanes == 2) go(std::integral_constant<int, 2>{}, vec_);
      else if (lanes == 4) go(std::integral_constant<int, 4>{}, vec_);
      else if (lanes == 8) go(std::integral_constant<int, 8>{}, vec_);
      else go(std::integral_constant<int, 16>{}, vec_);
    };
    if (vec) pick(std::true_type{});
    else pick(std::false_type{});
    QB_LAUNCH_OK("float_update_kernel");
    return QB_OK;
  });
}
