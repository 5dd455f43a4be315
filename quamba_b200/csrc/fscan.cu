// Selective scan in floating point with gradients, channel-last (sm_100a): the Mamba1 recurrence of a float model.
//
//   delta = softplus(dt + bias), h_t[n] = exp(delta_t A[n]) h_{t-1}[n] + delta_t x_t B_t[n], y_t = (C_t . h_t + D x_t) silu(z_t)
//
// A warp owns 512 states of one sequence: 8 groups of lanes x 4 lanes; the four lanes of a group share kCh channels and hold
// kNp consecutive states of each (kCh * kNp = 16 states a lane).  So the states' sums over n are shuffles between four lanes,
// what a token's B and C cost is one 128-bit read each for all channels of a lane, and in the backward pass the sums over
// channels (dB, dC) are taken in the lane first and then between eight lanes.  States and sums are float32 throughout, walked in
// packed pairs.
//
// Bound: dstate exponentials per (token, channel) on the MUFU pipe (16 results per clock and SM): 16 states cost 1 clock per
// (token, channel) and SM, while its bytes (8 at 16 bits) take 0.18 clocks of HBM time.
#include <algorithm>
#include "common.cuh"

namespace qb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kCkpt = 16;              // tokens between two kept states
constexpr int kRec = 512;              // states of a warp
constexpr int kSum = kRec + 32;        // a segment's summary: its states from zero, and the summed delta of its channels
constexpr int kGrad = kRec + 64;       // a warp's sums for dA | dD | d_bias
constexpr int kBwdWarps = 4;

template <typename T, int kNp_>
struct Geo {
  static constexpr int kNp = kNp_, kPairs = kNp / 2, kCh = 16 / kNp, kWc = 8 * kCh, kN = 4 * kNp;
  static constexpr int kLanesRow = kWc / 4;             // lanes that hold one token's channels, four each
  static constexpr int kRows = 32 / kLanesRow;          // tokens per warp-wide access
};

__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// max(v, 0) + log1p(e), e = exp(-|v|); log1p(e) = 2 artanh(s) with s = e / (2 + e) <= 1/3, by its series up to s^15 (the next
// term is below 2^-29 of the sum).
__device__ __forceinline__ float softplus_series(float v) {
  const float e = fast_exp2(-fabsf(v) * kLog2e);
  const float s = e * rcp_fast(2.0f + e), w = s * s;
  float p = fmaf(w, 1.0f / 15, 1.0f / 13);
  p = fmaf(w, p, 1.0f / 11);
  p = fmaf(w, p, 1.0f / 9);
  p = fmaf(w, p, 1.0f / 7);
  p = fmaf(w, p, 1.0f / 5);
  p = fmaf(w, p, 1.0f / 3);
  p = fmaf(w, p, 1.0f);
  return fmaf(2.0f * s, p, fmaxf(v, 0.0f));
}
__device__ __forceinline__ float sigmoid_fast(float v) {
  const float e = fast_exp2(-fabsf(v) * kLog2e), r = rcp_fast(1.0f + e);
  return v >= 0.0f ? r : e * r;
}
__device__ __forceinline__ f2 exp2_pair(f2 x) {
  float a, b;
  unpack2(x, a, b);
  return pack2(fast_exp2(a), fast_exp2(b));
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
    T v[4];
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
template <typename T>
__device__ __forceinline__ void stage_quad(T* dst, const T* src, int count, bool vec) {
  if (count <= 0) return;
  if (vec) {
    copy_async<4 * sizeof(T)>(dst, src);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < count) dst[k] = src[k];
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
  if constexpr (kCh == 4) {
    const float4 w = *reinterpret_cast<const float4*>(p);
    v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
  } else if constexpr (kCh == 2) {
    const float2 w = *reinterpret_cast<const float2*>(p);
    v[0] = w.x; v[1] = w.y;
  } else {
    v[0] = *p;
  }
}

// v[c] summed over the four lanes of a group; the lane gets the total of its own channel, q * kCh / 4
template <int kCh>
__device__ __forceinline__ float own_channel(const float (&v)[kCh], int q) {
  const bool hi = q & 2, odd = q & 1;
  if constexpr (kCh == 4) {
    const float a = (hi ? v[2] : v[0]) + __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[2], 2);
    const float b = (hi ? v[3] : v[1]) + __shfl_xor_sync(0xffffffffu, hi ? v[1] : v[3], 2);
    return (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
  } else if constexpr (kCh == 2) {
    const float a = (hi ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[1], 2);
    return a + __shfl_xor_sync(0xffffffffu, a, 1);
  } else {
    const float a = v[0] + __shfl_xor_sync(0xffffffffu, v[0], 2);
    return a + __shfl_xor_sync(0xffffffffu, a, 1);
  }
}

// where a warp stands
template <typename G>
struct Place {
  int lane, q, cg;
  int b, seg, ch0, nch, group, tile;                     // the tile's first channel and how many exist
  int own;                                               // the channel (of the tile) whose sums this lane gets
  bool writes;
  __device__ __forceinline__ Place(const qb_float_scan_args& a, int tpg, int b_, int seg_, int tile_, int lane_) {
    lane = lane_; q = lane & 3; cg = lane >> 2;
    b = b_; seg = seg_; tile = tile_;
    const int per = a.dim / a.groups;
    group = tile / tpg;
    const int c0 = (tile % tpg) * G::kWc;
    ch0 = group * per + c0;
    nch = min(G::kWc, per - c0);
    own = cg * G::kCh + q * G::kCh / 4;
    writes = q % (4 / G::kCh) == 0 && own < nch;
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
// the same in the library's own order, 16 bytes per lane and access
template <typename G, typename P>
__device__ __forceinline__ void load_record(const P* rec, int lane, f2 (&h)[G::kCh][G::kPairs]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const ulonglong2 v = *(reinterpret_cast<const ulonglong2*>(rec) + (i / 2) * 32 + lane);
    h[i / G::kPairs][i % G::kPairs] = v.x;
    h[(i + 1) / G::kPairs][(i + 1) % G::kPairs] = v.y;
  }
}
template <typename G, typename P>
__device__ __forceinline__ void store_record(P* rec, int lane, const f2 (&h)[G::kCh][G::kPairs]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    *(reinterpret_cast<ulonglong2*>(rec) + (i / 2) * 32 + lane) =
        make_ulonglong2(h[i / G::kPairs][i % G::kPairs], h[(i + 1) / G::kPairs][(i + 1) % G::kPairs]);
}
// h <- what the summarised segment makes of it
template <typename G>
__device__ __forceinline__ void fold(const float* sum, const Place<G>& w, const f2 (&A)[G::kCh][G::kPairs], f2 (&h)[G::kCh][G::kPairs]) {
  f2 loc[G::kCh][G::kPairs];
  load_record<G>(sum, w.lane, loc);
#pragma unroll
  for (int c = 0; c < G::kCh; ++c) {
    const float d = sum[kRec + w.cg * G::kCh + c];
#pragma unroll
    for (int p = 0; p < G::kPairs; ++p) h[c][p] = fma2(exp2_pair(mul2(pack2(d, d), A[c][p])), h[c][p], loc[c][p]);
  }
}

__device__ __forceinline__ int live_tokens(const qb_float_scan_args& a, int b) {
  return a.lengths != nullptr ? max(0, min(a.seqlen, a.lengths[b])) : a.seqlen;
}

// Raw rows of a tile of tokens, as they lie in memory.
template <typename T, typename G, int kT, int kWide>
struct Raw {
  T wide[kWide][kT][G::kWc];             // x, dt, z, dy
  T bc[2][kT][G::kN];
};
// stages tokens t0 .. min(t0 + kT, end) - 1
template <typename T, typename G, int kT, int kWide>
__device__ __forceinline__ void stage_tile(Raw<T, G, kT, kWide>& raw, const T* const (&src)[kWide], const int64_t (&stride)[kWide], const T* const (&bc)[2],
                                           const int64_t (&bc_stride)[2], int t0, int end, int nch, int dstate, bool vec, bool vec_bc, int lane) {
  const int row = lane / G::kLanesRow, c4 = (lane % G::kLanesRow) * 4;
#pragma unroll
  for (int i = 0; i < kT / G::kRows; ++i) {
    const int t = i * G::kRows + row;
    if (t0 + t < end) {
#pragma unroll
      for (int k = 0; k < kWide; ++k)
        if (src[k] != nullptr) stage_quad(&raw.wide[k][t][c4], src[k] + (int64_t)(t0 + t) * stride[k] + c4, nch - c4, vec);
    }
  }
  constexpr int kQuads = G::kN / 4;
#pragma unroll
  for (int i = 0; i < 2 * kT * kQuads / 32; ++i) {
    const int e = i * 32 + lane, n4 = (e % kQuads) * 4, t = (e / kQuads) % kT, k = e / kQuads / kT;
    if (t0 + t < end && bc[k] != nullptr) stage_quad(&raw.bc[k][t][n4], bc[k] + (int64_t)(t0 + t) * bc_stride[k] + n4, dstate - n4, vec_bc);
  }
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

struct Vec { int wide, bc; };

// ---- forward ----------------------------------------------------------------------------------------------------------------
template <typename T, typename G>
struct FwdSmem {
  static constexpr int kT = 16;
  Raw<T, G, kT, 3> raw[2];
  float delta[kT][G::kWc], u[kT][G::kWc];
  float bc[2][kT][G::kN];
};

// One warp: a tile of channels of one segment of one sequence.  kMode 0: outputs (from the folded summaries of the segments
// before); 1: the segment's summary; 2: the summary of the backward recurrence, from the segment's end to its start.
template <typename T, int kNp, int kMode>
__global__ void __launch_bounds__(32)
float_scan_kernel(const __grid_constant__ qb_float_scan_args a, int tpg, int nseg, int seg_len, float* sums, Vec vec) {
  using G = Geo<T, kNp>;
  using S = FwdSmem<T, G>;
  constexpr int kT = S::kT;
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
  if (kOut)
    for (int i = 0; i < w.seg; ++i) fold(sums + (((int64_t)w.b * nseg + i) * tiles + w.tile) * kSum, w, A, h);

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
  const float Dv = kOut && a.D != nullptr && w.own < w.nch ? a.D[w.ch0 + w.own] : 0.0f;
  const bool has_D = a.D != nullptr;
  T* const yp = kOut ? static_cast<T*>(a.y) + (int64_t)w.b * a.seqlen * a.dim + w.ch0 + w.own : nullptr;

  const int count = (int)((end - begin + kT - 1) / kT);
  auto tile_start = [&](int i) { return begin + (kRev ? count - 1 - i : i) * kT; };
  if (count > 0) stage_tile<T, G, kT, 3>(s.raw[0], src, stride, bc, bc_stride, tile_start(0), end, w.nch, a.dstate, vec.wide, vec.bc, lane);
  copy_commit();
  for (int i = 0; i < count; ++i) {
    const int t0 = tile_start(i);
    auto& raw = s.raw[i & 1];
    if (i + 1 < count) stage_tile<T, G, kT, 3>(s.raw[(i + 1) & 1], src, stride, bc, bc_stride, tile_start(i + 1), end, w.nch, a.dstate, vec.wide, vec.bc, lane);
    copy_commit();
    copy_wait<1>();
    __syncwarp();
    if (t0 < live) {
      if (kOut && a.checkpoints != nullptr && t0 > 0)
        store_record<G>(a.checkpoints + (((int64_t)w.b * ((a.seqlen + kCkpt - 1) / kCkpt) + t0 / kCkpt) * tiles + w.tile) * kRec, lane, h);
#pragma unroll
      for (int j = 0; j < kT / G::kRows; ++j) {
        const int t = j * G::kRows + row;
        const bool in = t0 + t < min(live, end);
        const float4 xv = quad(&raw.wide[0][t][c4]), dv = quad(&raw.wide[1][t][c4]);
        float4 zv;
        if (kRev && zp != nullptr) zv = quad(&raw.wide[2][t][c4]);
        float d[4], u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool on = in && c4 + k < w.nch;
          const float v = at(dv, k) + bias[k];
          d[k] = on ? (a.dt_softplus ? softplus_series(v) : v) : 0.0f;
          float g = at(xv, k);
          if (kRev) {
            if (zp != nullptr) g *= at(zv, k) * sigmoid_fast(at(zv, k));
          } else {
            g *= d[k];
          }
          u[k] = on ? g : 0.0f;
          sum[k] += d[k];
        }
        *reinterpret_cast<float4*>(&s.delta[t][c4]) = make_float4(d[0], d[1], d[2], d[3]);
        *reinterpret_cast<float4*>(&s.u[t][c4]) = make_float4(u[0], u[1], u[2], u[3]);
      }
      widen_bc<T, G, kT>(raw, s.bc, t0, min(live, end), a.dstate, lane);
      __syncwarp();
#pragma unroll 4
      for (int j = 0; j < kT; ++j) {
        const int t = kRev ? kT - 1 - j : j;
        float d[G::kCh], u[G::kCh], y[G::kCh];
        f2 in2[G::kPairs], c2[G::kPairs];
        load_channels<G::kCh>(&s.delta[t][w.cg * G::kCh], d);
        load_channels<G::kCh>(&s.u[t][w.cg * G::kCh], u);
        load_pairs<G::kPairs>(&s.bc[kRev ? 1 : 0][t][w.q * kNp], in2);
        if (kOut) load_pairs<G::kPairs>(&s.bc[1][t][w.q * kNp], c2);
#pragma unroll
        for (int c = 0; c < G::kCh; ++c) {
          const f2 dd = pack2(d[c], d[c]), uu = pack2(u[c], u[c]);
          f2 acc = 0ull;
#pragma unroll
          for (int p = 0; p < G::kPairs; ++p) {
            const f2 e = exp2_pair(mul2(dd, A[c][p]));
            if (kRev)
              h[c][p] = mul2(e, fma2(in2[p], uu, h[c][p]));
            else
              h[c][p] = fma2(e, h[c][p], mul2(in2[p], uu));
            if (kOut) acc = fma2(h[c][p], c2[p], acc);
          }
          if (kOut) {
            float lo, hi;
            unpack2(acc, lo, hi);
            y[c] = lo + hi;
          }
        }
        if (kOut) {
          float v = own_channel<G::kCh>(y, w.q);
          if (w.writes && t0 + t < end) {
            if (has_D) v = fmaf(Dv, to_f(raw.wide[0][t][w.own]), v);
            if (zp != nullptr) {
              const float zv = to_f(raw.wide[2][t][w.own]);
              v *= zv * sigmoid_fast(zv);
            }
            yp[(int64_t)(t0 + t) * a.dim] = from_f<T>(t0 + t < live ? v : 0.0f);
          }
        }
      }
    } else if (kOut && w.writes) {
      for (int t = t0; t < min(t0 + kT, end); ++t) yp[(int64_t)t * a.dim] = from_f<T>(0.0f);
    }
    __syncwarp();
  }
  if (kOut) {
    if (a.final_state != nullptr && w.seg == nseg - 1) store_state(a.final_state, a, w, h);
  } else {
    float* rec = sums + (((int64_t)w.b * nseg + w.seg) * tiles + w.tile) * kSum;
    store_record<G>(rec, lane, h);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int o = G::kLanesRow; o < 32; o <<= 1) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
      if (row == 0) rec[kRec + c4 + k] = sum[k];
    }
  }
}

// ---- backward ---------------------------------------------------------------------------------------------------------------
// With g_t = dy_t silu(z_t) and dh_t = C_t g_t + a_{t+1} dh_{t+1}:
//   dC_t = sum_d g_t h_t, dB_t = sum_d dh_t delta_t x_t, dx_t = delta_t sum_n dh_t B_t + D g_t,
//   ddelta_t = x_t sum_n dh_t B_t + sum_n A (dh_t a_t h_{t-1}), dA = sum_t delta_t (dh_t a_t h_{t-1}).
// A warp walks its segment's chunks of 16 tokens from the last to the first.  A chunk's states come from the one kept at its
// start: they are run forward once, and kept in shared memory before every fourth token; then four tokens at a time are run
// forward again with decays and states in registers, and walked back.  (Running all 16 back from registers needs 512 of them;
// keeping every state in shared memory moves 4 KB per token and warp through it.)
template <typename T, typename G>
struct BwdWarpSmem {
  static constexpr int kT = kCkpt;
  static constexpr int kBuf = sizeof(T) == 2 ? 2 : 1;
  Raw<T, G, kT, 4> raw[kBuf];
  float delta[kT][G::kWc], u[kT][G::kWc], g[kT][G::kWc];
  float bc[2][kT][G::kN];
  float keep[4][kRec];
  float part[kT][2][G::kN];
};

template <typename T, int kNp>
__global__ void __launch_bounds__(32 * kBwdWarps)
float_scan_bwd_kernel(const __grid_constant__ qb_float_scan_args a, int tpg, int nseg, int seg_len, const float* sums, float* part_bc, float* part_grad,
                      Vec vec) {
  using G = Geo<T, kNp>;
  using S = BwdWarpSmem<T, G>;
  constexpr int kT = S::kT, kBuf = S::kBuf, kV = 2 * kNp;
  extern __shared__ __align__(16) unsigned char dyn[];
  const int warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
  S& s = reinterpret_cast<S*>(dyn)[warp];
  const int cpg = (tpg + kBwdWarps - 1) / kBwdWarps, ctas = cpg * a.groups, tiles = tpg * a.groups;
  const int cta = (int)(blockIdx.x % ctas), rest = (int)(blockIdx.x / ctas);
  const int in_group = (cta % cpg) * kBwdWarps + warp;
  Place<G> w(a, tpg, rest / nseg, rest % nseg, (cta / cpg) * tpg + min(in_group, tpg - 1), lane);
  if (in_group >= tpg) {                                 // a warp past the group's last tile adds zeros to its CTA's sums
    w.nch = 0;
    w.writes = false;
  }
  const int live = live_tokens(a, w.b);
  const int begin = w.seg * seg_len, end = min(a.seqlen, begin + seg_len);

  f2 A[G::kCh][G::kPairs], carry[G::kCh][G::kPairs], dA[G::kCh][G::kPairs];
  load_A(a, w, A);
  load_state(a.d_final, a, w, carry);
  for (int i = nseg - 1; i > w.seg; --i) fold(sums + (((int64_t)w.b * nseg + i) * tiles + w.tile) * kSum, w, A, carry);
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
  const bool has_z = a.z != nullptr;
  const int row = lane / G::kLanesRow, c4 = (lane % G::kLanesRow) * 4;
  float bias[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) bias[k] = a.dt_bias != nullptr && c4 + k < w.nch ? a.dt_bias[w.ch0 + c4 + k] : 0.0f;
  const bool has_own = w.own < w.nch, has_D = a.D != nullptr;
  const float Dv = has_D && has_own ? a.D[w.ch0 + w.own] : 0.0f;
  const float own_bias = a.dt_bias != nullptr && has_own ? a.dt_bias[w.ch0 + w.own] : 0.0f;
  float dD = 0.0f, dbias = 0.0f;
  T* const dxp = a.d_x != nullptr ? static_cast<T*>(a.d_x) + at_out + w.own : nullptr;
  T* const ddp = a.d_dt != nullptr ? static_cast<T*>(a.d_dt) + at_out + w.own : nullptr;
  T* const dzp = a.d_z != nullptr && has_z ? static_cast<T*>(a.d_z) + at_out + w.own : nullptr;
  float* const part = part_bc + ((int64_t)cta * a.batch + w.b) * a.seqlen * (2 * G::kN);
  const int nck = (a.seqlen + kCkpt - 1) / kCkpt;

  const int first = begin / kT, last = (end + kT - 1) / kT - 1;
  // whole chunks past the sequence: zeros
  int chunk = last;
  for (; chunk >= first && chunk * kT >= live; --chunk) {
    const int lim = min(end, chunk * kT + kT);
    for (int t = chunk * kT; t < lim; ++t)
      if (w.writes) {
        if (dxp != nullptr) dxp[(int64_t)t * a.dim] = from_f<T>(0.0f);
        if (ddp != nullptr) ddp[(int64_t)t * a.dim] = from_f<T>(0.0f);
        if (dzp != nullptr) dzp[(int64_t)t * a.dim] = from_f<T>(0.0f);
      }
    for (int e = (int)threadIdx.x; e < (lim - chunk * kT) * 2 * G::kN; e += 32 * kBwdWarps) part[(int64_t)chunk * kT * 2 * G::kN + e] = 0.0f;
  }
  const int top = chunk;
  if (kBuf == 2) {
    if (top >= first) stage_tile<T, G, kT, 4>(s.raw[0], src, stride, bc, bc_stride, top * kT, end, w.nch, a.dstate, vec.wide, vec.bc, lane);
    copy_commit();
  }
  for (; chunk >= first; --chunk) {
    const int t0 = chunk * kT, lim = min(live, end);
    auto& raw = s.raw[(top - chunk) % kBuf];
    if (kBuf == 2) {
      if (chunk > first)
        stage_tile<T, G, kT, 4>(s.raw[(top - chunk + 1) % kBuf], src, stride, bc, bc_stride, t0 - kT, end, w.nch, a.dstate, vec.wide, vec.bc, lane);
      copy_commit();
      copy_wait<1>();
    } else {
      stage_tile<T, G, kT, 4>(raw, src, stride, bc, bc_stride, t0, end, w.nch, a.dstate, vec.wide, vec.bc, lane);
      copy_commit();
      copy_wait<0>();
    }
    f2 h[G::kCh][G::kPairs];
    if (chunk == 0)
      load_state(a.initial_state, a, w, h);
    else
      load_record<G>(a.checkpoints + (((int64_t)w.b * nck + chunk) * tiles + w.tile) * kRec, lane, h);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kT / G::kRows; ++j) {
      const int t = j * G::kRows + row;
      const bool in = t0 + t < lim;
      const float4 xv = quad(&raw.wide[0][t][c4]), dv = quad(&raw.wide[1][t][c4]), yv = quad(&raw.wide[3][t][c4]);
      float4 zv;
      if (has_z) zv = quad(&raw.wide[2][t][c4]);
      float d[4], u[4], g[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool on = in && c4 + k < w.nch;
        const float v = at(dv, k) + bias[k];
        d[k] = on ? (a.dt_softplus ? softplus_series(v) : v) : 0.0f;
        u[k] = on ? d[k] * at(xv, k) : 0.0f;
        float gg = at(yv, k);
        if (has_z) gg *= at(zv, k) * sigmoid_fast(at(zv, k));
        g[k] = on ? gg : 0.0f;
      }
      *reinterpret_cast<float4*>(&s.delta[t][c4]) = make_float4(d[0], d[1], d[2], d[3]);
      *reinterpret_cast<float4*>(&s.u[t][c4]) = make_float4(u[0], u[1], u[2], u[3]);
      *reinterpret_cast<float4*>(&s.g[t][c4]) = make_float4(g[0], g[1], g[2], g[3]);
    }
    widen_bc<T, G, kT>(raw, s.bc, t0, lim, a.dstate, lane);
    __syncwarp();
    // states before every fourth token
    store_record<G>(&s.keep[0][0], lane, h);
#pragma unroll 1
    for (int sub = 1; sub < 4; ++sub) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = (sub - 1) * 4 + j;
        float d[G::kCh], u[G::kCh];
        f2 b2[G::kPairs];
        load_channels<G::kCh>(&s.delta[t][w.cg * G::kCh], d);
        load_channels<G::kCh>(&s.u[t][w.cg * G::kCh], u);
        load_pairs<G::kPairs>(&s.bc[0][t][w.q * kNp], b2);
#pragma unroll
        for (int c = 0; c < G::kCh; ++c) {
          const f2 dd = pack2(d[c], d[c]), uu = pack2(u[c], u[c]);
#pragma unroll
          for (int p = 0; p < G::kPairs; ++p) h[c][p] = fma2(exp2_pair(mul2(dd, A[c][p])), h[c][p], mul2(b2[p], uu));
        }
      }
      store_record<G>(&s.keep[sub][0], lane, h);
    }
#pragma unroll 1
    for (int sub = 3; sub >= 0; --sub) {
      f2 e[4][G::kCh][G::kPairs], hp[5][G::kCh][G::kPairs];
      float inner[4];
      load_record<G>(&s.keep[sub][0], lane, hp[0]);      // a lane reads what it wrote itself
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = sub * 4 + j;
        float d[G::kCh], u[G::kCh], y[G::kCh];
        f2 b2[G::kPairs], c2[G::kPairs];
        load_channels<G::kCh>(&s.delta[t][w.cg * G::kCh], d);
        load_channels<G::kCh>(&s.u[t][w.cg * G::kCh], u);
        load_pairs<G::kPairs>(&s.bc[0][t][w.q * kNp], b2);
        load_pairs<G::kPairs>(&s.bc[1][t][w.q * kNp], c2);
#pragma unroll
        for (int c = 0; c < G::kCh; ++c) {
          const f2 dd = pack2(d[c], d[c]), uu = pack2(u[c], u[c]);
          f2 acc = 0ull;
#pragma unroll
          for (int p = 0; p < G::kPairs; ++p) {
            e[j][c][p] = exp2_pair(mul2(dd, A[c][p]));
            hp[j + 1][c][p] = fma2(e[j][c][p], hp[j][c][p], mul2(b2[p], uu));
            acc = fma2(hp[j + 1][c][p], c2[p], acc);
          }
          float lo, hi;
          unpack2(acc, lo, hi);
          y[c] = lo + hi;
        }
        inner[j] = has_z ? own_channel<G::kCh>(y, w.q) : 0.0f;
      }
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        const int t = sub * 4 + j;
        float d[G::kCh], u[G::kCh], g[G::kCh], through[G::kCh], into[G::kCh];
        f2 b2[G::kPairs], c2[G::kPairs], sB[G::kPairs], sC[G::kPairs];
        load_channels<G::kCh>(&s.delta[t][w.cg * G::kCh], d);
        load_channels<G::kCh>(&s.u[t][w.cg * G::kCh], u);
        load_channels<G::kCh>(&s.g[t][w.cg * G::kCh], g);
        load_pairs<G::kPairs>(&s.bc[0][t][w.q * kNp], b2);
        load_pairs<G::kPairs>(&s.bc[1][t][w.q * kNp], c2);
#pragma unroll
        for (int p = 0; p < G::kPairs; ++p) sB[p] = sC[p] = 0ull;
#pragma unroll
        for (int c = 0; c < G::kCh; ++c) {
          const f2 dd = pack2(d[c], d[c]), uu = pack2(u[c], u[c]), gg = pack2(g[c], g[c]);
          f2 thr = 0ull, q2 = 0ull;
#pragma unroll
          for (int p = 0; p < G::kPairs; ++p) {
            const f2 dh = fma2(c2[p], gg, carry[c][p]);
            sC[p] = fma2(gg, hp[j + 1][c][p], sC[p]);
            sB[p] = fma2(uu, dh, sB[p]);
            thr = fma2(dh, b2[p], thr);
            carry[c][p] = mul2(dh, e[j][c][p]);
            const f2 v = mul2(carry[c][p], hp[j][c][p]);
            q2 = fma2(v, A[c][p], q2);
            dA[c][p] = fma2(v, dd, dA[c][p]);
          }
          float lo, hi;
          unpack2(thr, lo, hi);
          through[c] = lo + hi;
          unpack2(q2, lo, hi);
          into[c] = lo + hi;
        }
        // dB and dC of this token over the warp's channels: value i of a lane's 2 kNp is (B | C, state); eight lane groups
        // halve the list three times
        float v[kV];
#pragma unroll
        for (int p = 0; p < G::kPairs; ++p) {
          unpack2(sB[p], v[2 * p], v[2 * p + 1]);
          unpack2(sC[p], v[kNp + 2 * p], v[kNp + 2 * p + 1]);
        }
#pragma unroll
        for (int half = kV / 2, bit = 16; bit >= 4; half /= 2, bit >>= 1) {
          const bool up = lane & bit;
#pragma unroll
          for (int k = 0; k < half; ++k) v[k] = (up ? v[half + k] : v[k]) + __shfl_xor_sync(0xffffffffu, up ? v[k] : v[half + k], bit);
        }
        const int at0 = ((lane >> 4) & 1) * (kV / 2) + ((lane >> 3) & 1) * (kV / 4) + ((lane >> 2) & 1) * (kV / 8);
#pragma unroll
        for (int k = 0; k < kV / 8; ++k) s.part[t][(at0 + k) / kNp][w.q * kNp + (at0 + k) % kNp] = v[k];

        const float own_through = own_channel<G::kCh>(through, w.q), own_into = own_channel<G::kCh>(into, w.q) * kLn2;
        if (w.writes && t0 + t < end) {
          const bool in = t0 + t < lim;
          const float xv = to_f(raw.wide[0][t][w.own]), dl = s.delta[t][w.own], gv = s.g[t][w.own];
          const float dx = fmaf(Dv, gv, own_through * dl);
          float dd = fmaf(own_through, xv, own_into);
          if (a.dt_softplus) dd *= sigmoid_fast(to_f(raw.wide[1][t][w.own]) + own_bias);
          const int64_t o = (int64_t)(t0 + t) * a.dim;
          if (in) {
            dD = fmaf(gv, xv, dD);
            dbias += dd;
          }
          if (dxp != nullptr) dxp[o] = from_f<T>(in ? dx : 0.0f);
          if (ddp != nullptr) ddp[o] = from_f<T>(in ? dd : 0.0f);
          if (dzp != nullptr) {
            const float zv = to_f(raw.wide[2][t][w.own]), sig = sigmoid_fast(zv);
            float all = inner[j];
            if (has_D) all = fmaf(Dv, xv, all);
            dzp[o] = from_f<T>(in ? to_f(raw.wide[3][t][w.own]) * all * sig * fmaf(zv, 1.0f - sig, 1.0f) : 0.0f);
          }
        }
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
    float* rec = part_grad + (((int64_t)w.b * nseg + w.seg) * tiles + w.tile) * kGrad;
    store_record<G>(rec, lane, dA);
    if (w.writes) {
      rec[kRec + w.own] = dD;
      rec[kRec + 32 + w.own] = dbias;
    }
    if (a.d_initial != nullptr && w.seg == 0) store_state(a.d_initial, a, w, carry);
  }
}

// dB and dC: the CTAs' sums added up in their order
template <typename T>
__global__ void __launch_bounds__(256) float_scan_bc_kernel(const __grid_constant__ qb_float_scan_args a, const float* part, int cpg, int npad) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;      // (b, t, group, B | C, n)
  const int n = (int)(i % npad), k = (int)(i / npad % 2), g = (int)(i / (2 * npad) % a.groups);
  const int64_t bt = i / ((int64_t)2 * npad * a.groups), tokens = (int64_t)a.batch * a.seqlen;
  if (bt >= tokens || n >= a.dstate) return;
  const float* p = part + ((int64_t)g * cpg * tokens + bt) * (2 * npad) + k * npad + n;
  float v = 0.0f;
  for (int c = 0; c < cpg; ++c) v += p[(int64_t)c * tokens * (2 * npad)];
  T* out = static_cast<T*>(k ? a.d_C : a.d_B);
  if (out != nullptr) out[(bt * a.groups + g) * a.dstate + n] = from_f<T>(v);
}

// dA, dD, d_bias: summed over sequences and segments in their order
template <int kNp>
__global__ void __launch_bounds__(kGrad) float_scan_param_kernel(const __grid_constant__ qb_float_scan_args a, const float* part, int tpg, int runs) {
  using G = Geo<float, kNp>;
  const int tiles = tpg * a.groups, tile = (int)blockIdx.x, i = (int)threadIdx.x;
  const int per = a.dim / a.groups, c0 = (tile % tpg) * G::kWc, ch0 = tile / tpg * per + c0, nch = min(G::kWc, per - c0);
  const bool is_A = i < kRec;
  // a record's float4 k of lane l holds the values 4 k .. 4 k + 3 of that lane, value = channel of the lane * kNp + state
  const int l = i / 4 % 32, v = i / 128 * 4 + i % 4;
  const int ch = is_A ? (l >> 2) * G::kCh + v / kNp : (i - kRec) % 32, n = is_A ? (l & 3) * kNp + v % kNp : 0;
  if (ch >= nch || (is_A && n >= a.dstate)) return;
  const float* p = part + (int64_t)tile * kGrad + i;
  float sum = 0.0f;
  for (int r = 0; r < runs; ++r) sum += p[(int64_t)r * tiles * kGrad];
  if (is_A) {
    if (a.d_A != nullptr) a.d_A[(int64_t)(ch0 + ch) * a.dstate + n] = sum;
  } else if (i < kRec + 32) {
    if (a.d_D != nullptr) a.d_D[ch0 + ch] = sum;
  } else if (a.d_bias != nullptr) {
    a.d_bias[ch0 + ch] = sum;
  }
}

// ---- one token --------------------------------------------------------------------------------------------------------------
// Bound by the state, read and written once (8 bytes per state).  kLanes lanes of a channel hold four states each.
template <typename T, int kLanes>
__global__ void __launch_bounds__(128) float_update_kernel(const __grid_constant__ qb_float_update_args a, int vec) {
  const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
  const int sub = (int)(i % kLanes), n0 = sub * 4;
  const int64_t bd = min(i / kLanes, (int64_t)a.batch * a.dim - 1);      // the last lanes repeat the last channel, for the shuffles
  const bool mine = i / kLanes == bd;
  const int b = (int)(bd / a.dim), d = (int)(bd % a.dim), g = d / (a.dim / a.groups);
  const float* st = a.state + b * a.state_sb + (int64_t)d * a.state_sd + n0;
  float h[4], A[4], B[4], C[4];
  if (vec) {
    const float4 v = n0 < a.dstate ? *reinterpret_cast<const float4*>(st) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    h[0] = v.x; h[1] = v.y; h[2] = v.z; h[3] = v.w;
  }
  const T* Bp = static_cast<const T*>(a.Bm) + b * a.B_sb + (int64_t)g * a.B_sg + n0;
  const T* Cp = static_cast<const T*>(a.Cm) + b * a.C_sb + (int64_t)g * a.C_sg + n0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const bool in = n0 + k < a.dstate;
    if (!vec) h[k] = in ? st[k] : 0.0f;
    A[k] = in ? a.A[(int64_t)d * a.dstate + n0 + k] * kLog2e : 0.0f;
    B[k] = in ? to_f(Bp[k]) : 0.0f;
    C[k] = in ? to_f(Cp[k]) : 0.0f;
  }
  const float x = to_f(static_cast<const T*>(a.x)[b * a.x_sb + d]);
  float dl = to_f(static_cast<const T*>(a.dt)[b * a.dt_sb + d]) + (a.dt_bias != nullptr ? a.dt_bias[d] : 0.0f);
  if (a.dt_softplus) dl = softplus_series(dl);
  const float u = dl * x;
  float y = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    h[k] = fmaf(fast_exp2(dl * A[k]), h[k], u * B[k]);
    y = fmaf(h[k], C[k], y);
  }
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  if (!mine) return;
  float* so = a.state_out + b * a.state_out_sb + (int64_t)d * a.state_out_sd + n0;
  if (vec) {
    if (n0 < a.dstate) *reinterpret_cast<float4*>(so) = make_float4(h[0], h[1], h[2], h[3]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n0 + k < a.dstate) so[k] = h[k];
  }
  if (sub == 0) {
    if (a.D != nullptr) y = fmaf(a.D[d], x, y);
    if (a.z != nullptr) {
      const float z = to_f(static_cast<const T*>(a.z)[b * a.z_sb + d]);
      y *= z * sigmoid_fast(z);
    }
    static_cast<T*>(a.y)[(int64_t)b * a.dim + d] = from_f<T>(y);
  }
}

// ---- host -------------------------------------------------------------------------------------------------------------------
struct Plan {
  int np, wc, tpg, tiles, nseg, seg_len;
};
Plan plan_of(int batch, int seqlen, int dim, int groups, int dstate) {
  Plan p;
  p.np = dstate <= 16 ? 4 : dstate <= 32 ? 8 : 16;
  p.wc = 128 / p.np;
  p.tpg = (int)ceil_div(dim / groups, p.wc);
  p.tiles = p.tpg * groups;
  p.nseg = 1;
  p.seg_len = std::max(seqlen, 1);
  (void)batch;
  return p;
}
int64_t align256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t sums_bytes(const Plan& p, int64_t batch) { return p.nseg > 1 ? align256(batch * p.nseg * p.tiles * kSum * (int64_t)sizeof(float)) : 0; }
int64_t part_bytes(const Plan& p, int64_t batch, int64_t seqlen, int groups) {
  return align256(ceil_div(p.tpg, kBwdWarps) * groups * batch * seqlen * 8 * p.np * (int64_t)sizeof(float));
}
int64_t grad_bytes(const Plan& p, int64_t batch) { return align256(batch * p.nseg * p.tiles * kGrad * (int64_t)sizeof(float)); }

bool sizes_ok(int64_t batch, int64_t seqlen, int64_t dim, int64_t groups, int64_t dstate) {
  return batch >= 0 && seqlen >= 0 && dim > 0 && groups > 0 && dim % groups == 0 && dstate >= 1 && dstate <= 64;
}
bool quads(const void* p, int64_t s1, int64_t s2, size_t size) { return p == nullptr || (aligned(p, 4 * size) && s1 % 4 == 0 && s2 % 4 == 0); }

int check_scan(const qb_float_scan_args* a, const char* who) {
  QB_REQUIRE(a != nullptr && a->x && a->dt && a->Bm && a->Cm && a->A, QB_ERR_INVALID_ARG, "%s: null pointer", who);
  QB_REQUIRE(a->dstate >= 1 && a->dstate <= 64, QB_ERR_INVALID_ARG, "%s: dstate must be 1 to 64, got %d", who, a->dstate);
  QB_REQUIRE(a->batch >= 0 && a->seqlen >= 0 && a->dim > 0 && a->groups > 0, QB_ERR_INVALID_ARG, "%s: bad shape", who);
  QB_REQUIRE(a->dim % a->groups == 0, QB_ERR_INVALID_ARG, "%s: dim = %d is not divisible by groups = %d", who, a->dim, a->groups);
  QB_REQUIRE(a->dtype >= 0 && a->dtype <= 2, QB_ERR_INVALID_ARG, "%s: unsupported type", who);
  const Plan p = plan_of(a->batch, a->seqlen, a->dim, a->groups, a->dstate);
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

template <typename T, int kNp, int kMode>
int launch_scan(const qb_float_scan_args& a, const Plan& p, float* sums, Vec vec, cudaStream_t st) {
  const size_t smem = sizeof(FwdSmem<T, Geo<T, kNp>>);
  static PerDeviceOnce attr;
  const int rc = attr.run([&]() -> int {
    QB_CUDA_OK(cudaFuncSetAttribute(float_scan_kernel<T, kNp, kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    return QB_OK;
  });
  if (rc != QB_OK) return rc;
  const int64_t grid = (int64_t)a.batch * (p.nseg - (kMode == 0 ? 0 : 1)) * p.tiles;
  float_scan_kernel<T, kNp, kMode><<<(unsigned)grid, 32, smem, st>>>(a, p.tpg, p.nseg, p.seg_len, sums, vec);
  QB_LAUNCH_OK("float_scan_kernel");
  return QB_OK;
}

template <typename T, int kNp>
int run_fwd(const qb_float_scan_args& a, const Plan& p, cudaStream_t st) {
  float* sums = static_cast<float*>(a.workspace);
  const Vec vec = vec_of(a, false);
  if (p.nseg > 1) {
    const int rc = launch_scan<T, kNp, 1>(a, p, sums, vec, st);
    if (rc != QB_OK) return rc;
  }
  return launch_scan<T, kNp, 0>(a, p, sums, vec, st);
}

template <typename T, int kNp>
int run_bwd(const qb_float_scan_args& a, const Plan& p, cudaStream_t st) {
  using G = Geo<T, kNp>;
  unsigned char* ws = static_cast<unsigned char*>(a.workspace);
  float* sums = reinterpret_cast<float*>(ws);
  float* part = reinterpret_cast<float*>(ws + sums_bytes(p, a.batch));
  float* grad = reinterpret_cast<float*>(ws + sums_bytes(p, a.batch) + part_bytes(p, a.batch, a.seqlen, a.groups));
  const Vec vec = vec_of(a, true);
  if (p.nseg > 1 && a.batch > 0) {
    const int rc = launch_scan<T, kNp, 2>(a, p, sums, vec, st);
    if (rc != QB_OK) return rc;
  }
  const size_t smem = sizeof(BwdWarpSmem<T, G>) * kBwdWarps;
  static PerDeviceOnce attr;
  const int rc = attr.run([&]() -> int {
    QB_CUDA_OK(cudaFuncSetAttribute(float_scan_bwd_kernel<T, kNp>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    return QB_OK;
  });
  if (rc != QB_OK) return rc;
  const int cpg = (int)ceil_div(p.tpg, kBwdWarps);
  if (a.batch > 0) {
    const int64_t grid = (int64_t)a.batch * p.nseg * cpg * a.groups;
    float_scan_bwd_kernel<T, kNp><<<(unsigned)grid, 32 * kBwdWarps, smem, st>>>(a, p.tpg, p.nseg, p.seg_len, sums, part, grad, vec);
    QB_LAUNCH_OK("float_scan_bwd_kernel");
  }
  const int64_t cells = (int64_t)a.batch * a.seqlen * a.groups * 2 * G::kN;
  if (cells > 0 && (a.d_B != nullptr || a.d_C != nullptr)) {
    float_scan_bc_kernel<T><<<(unsigned)ceil_div(cells, 256), 256, 0, st>>>(a, part, cpg, G::kN);
    QB_LAUNCH_OK("float_scan_bc_kernel");
  }
  if (a.d_A != nullptr || a.d_D != nullptr || a.d_bias != nullptr) {
    float_scan_param_kernel<kNp><<<(unsigned)p.tiles, kGrad, 0, st>>>(a, grad, p.tpg, a.batch * p.nseg);
    QB_LAUNCH_OK("float_scan_param_kernel");
  }
  return QB_OK;
}

template <typename F>
int by_type(int dtype, F f) {
  return dtype == 0 ? f(float{}) : dtype == 1 ? f(__half{}) : f(__nv_bfloat16{});
}

}  // namespace
}  // namespace qb

using namespace qb;

extern "C" int64_t qb_float_scan_checkpoint_bytes(int32_t batch, int32_t seqlen, int32_t dim, int32_t groups, int32_t dstate) {
  if (!sizes_ok(batch, seqlen, dim, groups, dstate)) return -1;
  return (int64_t)batch * ceil_div(seqlen, kCkpt) * plan_of(batch, seqlen, dim, groups, dstate).tiles * kRec * (int64_t)sizeof(float);
}

extern "C" int64_t qb_float_scan_workspace_bytes(int32_t batch, int32_t seqlen, int32_t dim, int32_t groups, int32_t dstate, int32_t backward) {
  if (!sizes_ok(batch, seqlen, dim, groups, dstate)) return -1;
  const Plan p = plan_of(batch, seqlen, dim, groups, dstate);
  return sums_bytes(p, batch) + (backward ? part_bytes(p, batch, seqlen, groups) + grad_bytes(p, batch) : 0);
}

extern "C" int qb_float_scan_fwd(const qb_float_scan_args* a, void* stream) {
  const int rc = check_scan(a, "float_scan_fwd");
  if (rc != QB_OK) return rc;
  QB_REQUIRE(a->y != nullptr || (int64_t)a->batch * a->seqlen == 0, QB_ERR_INVALID_ARG, "float_scan_fwd: null output");
  if (a->batch == 0) return QB_OK;
  const Plan p = plan_of(a->batch, a->seqlen, a->dim, a->groups, a->dstate);
  const int64_t need = sums_bytes(p, a->batch);
  QB_REQUIRE(need == 0 || (a->workspace != nullptr && a->workspace_bytes >= need && aligned(a->workspace, 16)), QB_ERR_INVALID_ARG,
             "float_scan_fwd: the workspace must have %lld bytes, 16-byte aligned", (long long)need);
  QB_REQUIRE(aligned(a->checkpoints, 16), QB_ERR_INVALID_ARG, "float_scan_fwd: checkpoints must be 16-byte aligned");
  return by_type(a->dtype, [&](auto t) -> int {
    using T = decltype(t);
    cudaStream_t st = (cudaStream_t)stream;
    return p.np == 4 ? run_fwd<T, 4>(*a, p, st) : p.np == 8 ? run_fwd<T, 8>(*a, p, st) : run_fwd<T, 16>(*a, p, st);
  });
}

extern "C" int qb_float_scan_bwd(const qb_float_scan_args* a, void* stream) {
  const int rc = check_scan(a, "float_scan_bwd");
  if (rc != QB_OK) return rc;
  QB_REQUIRE((a->dy != nullptr && a->checkpoints != nullptr) || (int64_t)a->batch * a->seqlen == 0, QB_ERR_INVALID_ARG, "float_scan_bwd: dy and checkpoints are needed");
  QB_REQUIRE(aligned(a->checkpoints, 16), QB_ERR_INVALID_ARG, "float_scan_bwd: checkpoints must be 16-byte aligned");
  const Plan p = plan_of(a->batch, a->seqlen, a->dim, a->groups, a->dstate);
  const int64_t need = qb_float_scan_workspace_bytes(a->batch, a->seqlen, a->dim, a->groups, a->dstate, 1);
  QB_REQUIRE(need == 0 || (a->workspace != nullptr && a->workspace_bytes >= need && aligned(a->workspace, 16)), QB_ERR_INVALID_ARG,
             "float_scan_bwd: the workspace must have %lld bytes, 16-byte aligned", (long long)need);
  return by_type(a->dtype, [&](auto t) -> int {
    using T = decltype(t);
    cudaStream_t st = (cudaStream_t)stream;
    return p.np == 4 ? run_bwd<T, 4>(*a, p, st) : p.np == 8 ? run_bwd<T, 8>(*a, p, st) : run_bwd<T, 16>(*a, p, st);
  });
}

extern "C" int qb_float_scan_update(const qb_float_update_args* a, void* stream) {
  QB_REQUIRE(a != nullptr && a->state && a->state_out && a->x && a->dt && a->Bm && a->Cm && a->A && a->y, QB_ERR_INVALID_ARG, "float_scan_update: null pointer");
  QB_REQUIRE(sizes_ok(a->batch, 1, a->dim, a->groups, a->dstate), QB_ERR_INVALID_ARG,
             "float_scan_update: bad shape (dstate 1 to 64, dim divisible by groups)");
  QB_REQUIRE(a->dtype >= 0 && a->dtype <= 2, QB_ERR_INVALID_ARG, "float_scan_update: unsupported type");
  if (a->batch == 0) return QB_OK;
  const int lanes = a->dstate <= 4 ? 1 : a->dstate <= 8 ? 2 : a->dstate <= 16 ? 4 : a->dstate <= 32 ? 8 : 16;
  const int64_t grid = ceil_div((int64_t)a->batch * a->dim * lanes, 128);
  QB_REQUIRE(grid < (1ll << 31), QB_ERR_TOO_LARGE, "float_scan_update: batch and dim are too large");
  const int vec = a->dstate % 4 == 0 && aligned(a->state, 16) && aligned(a->state_out, 16) &&
                  (a->state_sb | a->state_sd | a->state_out_sb | a->state_out_sd) % 4 == 0;
  return by_type(a->dtype, [&](auto t) -> int {
    using T = decltype(t);
    cudaStream_t st = (cudaStream_t)stream;
    const unsigned g = (unsigned)grid;
    switch (lanes) {
      case 1: float_update_kernel<T, 1><<<g, 128, 0, st>>>(*a, vec); break;
      case 2: float_update_kernel<T, 2><<<g, 128, 0, st>>>(*a, vec); break;
      case 4: float_update_kernel<T, 4><<<g, 128, 0, st>>>(*a, vec); break;
      case 8: float_update_kernel<T, 8><<<g, 128, 0, st>>>(*a, vec); break;
      default: float_update_kernel<T, 16><<<g, 128, 0, st>>>(*a, vec);
    }
    QB_LAUNCH_OK("float_update_kernel");
    return QB_OK;
  });
}
