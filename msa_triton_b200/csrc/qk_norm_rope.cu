// RMS norm of every query and key head with the position rotation in the same pass,
// forward and backward: the step between a layer's projections and the index score /
// attention kernels (the reference takes unit-RMS rotated heads as given).
//
//   r = (mean(x^2) + eps)^(-1/2)       x' = x r        y = R(p) (w * x')
//   g' = R(p)^T g    dw = sum over tokens and heads of g' * x'    u = w * g'
//   dx = r (u - x' mean(u * x'))
//
// x is a head row of D elements of token t at position p; R(p) rotates the pairs of the
// first `rotary` elements by a table row of cosines and sines. All arithmetic is in
// float32; outputs and gradients are rounded once, when they are stored.
//
// HBM-bound (about one operation per byte): each row is read once, held in registers for the
// reduction and the rotation, and written once; the backward recomputes r from x (4 flops
// an element) instead of storing it. What is left to watch is the number of instructions: a warp has some 340
// issue slots to the 2 KB of rows that it reads and writes in the forward. So arithmetic is done two floats at a
// time, w and the angles are multiplied once for all the heads of a token, and addresses advance by a fixed
// step. Warps stay and walk over their tokens' heads, and hide one another's loads (a second set of registers for
// the next rows costs more warps than it gains: 243 against 210 us forward). q and k go through one launch, each
// with blocks of its own. The weights' gradients are summed in registers on the way, then over a block's warps and
// the blocks in a fixed order (no atomics, the same bits every run).
// Measured on the device: 32768 tokens of 64 + 8 heads of 128, bf16: 210 us forward, 5.8 TB/s, 90% of the copy rate;
// 71168 tokens of 32 + 8 heads: 256 us forward (88%), 407 us backward (5.4 TB/s, 83%).
#include <algorithm>

#include "rope_common.cuh"

namespace msa {
namespace {

using namespace rope;

constexpr int kWarps = 4;
constexpr int kMaxDimFast = 256;
constexpr int kMaxDim = 512;

// Rows a lane takes at a time: 64 bytes of loads in flight a tensor for every type.
template <typename T>
constexpr int kRowsOf = 64 / (2 * kE * (int)sizeof(T));

// Blocks to an SM, by registers (80 forward, 122 backward). Measured at 71168 tokens of 40 heads of 128: forward 256
// us with 6 blocks, 286 with 5; backward 407 us with 4, 427 with 5 and half the rows at a time, 465 with 7.
template <bool BWD>
constexpr int kResident = BWD ? 4 : 6;

// One of q and k.
struct Side {
  const void* x;
  const void* w;
  const void* g;  // backward: gradient of the output
  void* out;      // forward: y; backward: dx (may be null)
  int64_t x_ts, x_hs, g_ts, g_hs;  // strides in elements
  int heads;
  // A warp takes `slots` rows at a time: heads of one token, `chunks` steps a token. An item of work is `span`
  // steps of a token one after the other (`spans` items a token); the angles are loaded once for them. Where a
  // token's heads would not fill a warp (flat), it takes that many rows in a row whatever their tokens.
  uint32_t items, chunks, span, spans, first_block, blocks;
  bool flat;
};

struct Params {
  Side side[2];
  const float* table;
  const int32_t* positions;  // or null: from cu
  const int32_t* cu;
  float* partial;  // backward: [gridDim.x][dim] (any shape: [gridDim.x][2][dim]), or null
  int64_t table_rows, tokens;
  int nseq, dim, rotary, w_dtype;
  float eps, inv_dim;
  bool interleaved;
};

// Positions of tokens; the bounds of the last token's sequence are kept, so that a walk over the tokens
// searches once a sequence (a search is a chain of dependent loads ahead of the table's row).
struct Positions {
  int64_t lo = 0, hi = 0;
  __device__ __forceinline__ int64_t of(const Params& p, int64_t t) {
    if (p.positions) return p.positions[t];
    if (t < lo || t >= hi) {
      const int s = find_sequence(p.cu, p.nseq, t);
      lo = p.cu[s], hi = p.cu[s + 1];
    }
    return t - lo;
  }
};

__device__ __forceinline__ float load_weight(const void* w, int i, int dtype) {
  if (dtype == MSA_F32) return reinterpret_cast<const float*>(w)[i];
  if (dtype == MSA_F16) return __half2float(reinterpret_cast<const __half*>(w)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[i]);
}

template <bool INTER>
__device__ __forceinline__ Lane weights_of(const void* w, int dtype, const LaneMap& m) {
  float a[kE], b[kE], v[2 * kE];
#pragma unroll
  for (int i = 0; i < kE; ++i) a[i] = load_weight(w, m.a + i, dtype), b[i] = load_weight(w, m.b + i, dtype);
  to_pairs<INTER>(a, b, v);
  return lane_of(v);
}

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// ------------------------------------------------------------------ rows in the lane layout
// A lane's angles of one position, kE cosines and sines; lanes behind the rotated elements: 1 and 0.
struct Angles {
  float c[kE] = {1.f, 1.f, 1.f, 1.f}, s[kE] = {};
  bool inside = true;
  __device__ __forceinline__ void load(const Params& p, Positions& positions, const LaneMap& m, int64_t t, int l) {
    const int64_t pos = positions.of(p, t);
    inside = pos >= 0 && pos < p.table_rows;
#pragma unroll
    for (int i = 0; i < kE; ++i) c[i] = 1.f, s[i] = 0.f;
    if (inside && m.rotated) load_angles(p.table + pos * p.rotary, p.rotary, l, c, s);
  }
};

// The forward rotation of w * x, of a pair's x = (a, b): (a c0 + b s1, b c1 + a s0).
struct Turn {
  F2 c0[kE / 2], s1[kE / 2], c1[kE / 2], s0[kE / 2];
  __device__ __forceinline__ Turn(const Angles& t, const Lane& w) {
#pragma unroll
    for (int i = 0; i < kE / 2; ++i) {
      const F2 c = pack2(t.c[2 * i], t.c[2 * i + 1]), s = pack2(t.s[2 * i], t.s[2 * i + 1]);
      c0[i] = mul2(c, w.v[i]), s0[i] = mul2(s, w.v[i]);
      c1[i] = mul2(c, w.v[kE / 2 + i]);
      s1[i] = mul2(pack2(-t.s[2 * i], -t.s[2 * i + 1]), w.v[kE / 2 + i]);
    }
  }
};

// y of one row.
template <int LPR, bool INTER>
__device__ __forceinline__ void fwd_row(const Params& p, const LaneMap& m, const float (&f)[2 * kE], const Lane& w,
                                        uint32_t t, int l, bool inside, const Turn& turn, float (&out)[2 * kE]) {
  const Lane x = lane_of(f);
  const float ss = row_sum<LPR>(dot_of(x, x));
  const float r = inside ? rsqrtf(ss * p.inv_dim + p.eps) : nan_f32();
  const F2 rr = twice(r);
  Lane y;
#pragma unroll
  for (int e = 0; e < kE / 2; ++e) {
    y.v[e] = mul2(rr, fma2(x.v[e], turn.c0[e], mul2(x.v[kE / 2 + e], turn.s1[e])));
    y.v[kE / 2 + e] = mul2(rr, fma2(x.v[kE / 2 + e], turn.c1[e], mul2(x.v[e], turn.s0[e])));
  }
  floats_of(y, out);
  if (!(ss < INFINITY)) {  // an infinite or NaN row: element by element, as the formula has it
    float g[2 * kE];
    floats_of(w, g);
#pragma unroll
    for (int e = 0; e < 2 * kE; ++e) out[e] = f[e] * r * g[e];
    if (m.rotated) {
      Positions positions;
      Angles again;
      again.load(p, positions, m, t, l);
      rotate_lane(out, again.c, again.s);
    }
  }
}

// dx of one row, and its part of dw.
template <int LPR>
__device__ __forceinline__ void bwd_row(const Params& p, const LaneMap& m, const Lane& x, const Lane& g,
                                        const Lane& w, const Angles& t, bool counts, Lane& dw,
                                        float (&out)[2 * kE]) {
  // u = R^T g, the transposed rotation; part = u x element by element
  Lane u = g, part;
  if (m.rotated) {
#pragma unroll
    for (int e = 0; e < kE / 2; ++e) {
      const F2 c = pack2(t.c[2 * e], t.c[2 * e + 1]), s = pack2(t.s[2 * e], t.s[2 * e + 1]),
               minus = pack2(-t.s[2 * e], -t.s[2 * e + 1]);
      u.v[e] = fma2(g.v[e], c, mul2(g.v[kE / 2 + e], s));
      u.v[kE / 2 + e] = fma2(g.v[kE / 2 + e], c, mul2(g.v[e], minus));
    }
  }
#pragma unroll
  for (int e = 0; e < kE; ++e) part.v[e] = mul2(u.v[e], x.v[e]);
  // mean(w u x') = r mean(w u x): both sums from the row as it was read
  const float ss = row_sum<LPR>(dot_of(x, x)), dot = row_sum<LPR>(dot_of(part, w));
  const float r = t.inside ? rsqrtf(ss * p.inv_dim + p.eps) : nan_f32();
  const F2 rr = twice(r), minus_k = twice(-(dot * r * p.inv_dim * r * r));  // dx = r w u - k x
  const F2 count = counts ? rr : twice(0.f);
  Lane y;
#pragma unroll
  for (int e = 0; e < kE; ++e) {
    if (counts) dw.v[e] = fma2(part.v[e], count, dw.v[e]);
    y.v[e] = fma2(mul2(u.v[e], w.v[e]), rr, mul2(x.v[e], minus_k));
  }
  floats_of(y, out);
}

// The rows of a step: heads h, h + SUB, ... below `end`, each lane's two runs.
template <typename T, int ROWS, int SUB>
__device__ __forceinline__ void fetch(const T* row, int64_t hs, const LaneMap& m, int h, int end,
                                      Raw<T> (&raw)[ROWS][2]) {
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    raw[i][0].u = raw[i][1].u = {};
    if (m.active && h + i * SUB < end) {
      raw[i][0] = load_run(row + m.a);
      raw[i][1] = load_run(row + m.b);
    }
    row += SUB * hs;
  }
}

template <typename T, int LPR, bool INTER>
__global__ void __launch_bounds__(kWarps * 32, kResident<false>) fwd_kernel(const __grid_constant__ Params p) {
  constexpr int kRows = kRowsOf<T>, kSub = 32 / LPR, kSlots = kSub * kRows;
  const Side& s = p.side[blockIdx.x >= p.side[1].first_block];
  const int lane = threadIdx.x & 31, l = lane % LPR, sub = lane / LPR;
  const LaneMap m = lane_map<INTER>(l, p.dim, p.rotary);
  const uint32_t first = (blockIdx.x - s.first_block) * kWarps + (threadIdx.x >> 5), stride = s.blocks * kWarps;
  Lane w{};
  if (m.active) w = weights_of<INTER>(s.w, p.w_dtype, m);
  T* const out = static_cast<T*>(s.out);
  Positions positions;
  if (s.flat) {
    const uint32_t rows = (uint32_t)p.tokens * s.heads;
    for (uint32_t item = first; item < s.items; item += stride) {
      Raw<T> raw[kRows][2];
      uint32_t token[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const uint32_t row = item * kSlots + i * kSub + sub, t = row / (uint32_t)s.heads;
        token[i] = t;
        raw[i][0].u = raw[i][1].u = {};
        if (row < rows && m.active) {
          const T* x = static_cast<const T*>(s.x) + t * s.x_ts + (row - t * s.heads) * s.x_hs;
          raw[i][0] = load_run(x + m.a), raw[i][1] = load_run(x + m.b);
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const uint32_t row = item * kSlots + i * kSub + sub, t = token[i];
        const bool ok = row < rows && m.active;
        Angles angles;
        if (ok) angles.load(p, positions, m, t, l);
        float f[2 * kE], y[2 * kE];
        unpack_lane<INTER>(raw[i], f);
        fwd_row<LPR, INTER>(p, m, f, w, t, l, angles.inside, Turn(angles, w), y);
        if (ok) store_lane<INTER>(out + (int64_t)row * p.dim + m.a, out + (int64_t)row * p.dim + m.b, y);
      }
    }
    return;
  }
  for (uint32_t item = first; item < s.items; item += stride) {
    const uint32_t t = item / s.spans, chunk = (item - t * s.spans) * s.span;
    int h = (int)chunk * kSlots + sub;
    const int end = min((int)(chunk + s.span) * kSlots, s.heads);
    const T* x = static_cast<const T*>(s.x) + (int64_t)t * s.x_ts + h * s.x_hs;
    T* to = out + ((int64_t)t * s.heads + h) * p.dim;
    Raw<T> raw[kRows][2];
    fetch<T, kRows, kSub>(x, s.x_hs, m, h, end, raw);
    Angles angles;
    angles.load(p, positions, m, t, l);
    const Turn turn(angles, w);
    const bool inside = angles.inside;
    while (true) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        float f[2 * kE], y[2 * kE];
        unpack_lane<INTER>(raw[i], f);
        fwd_row<LPR, INTER>(p, m, f, w, t, l, inside, turn, y);
        if (h + i * kSub < end && m.active) store_lane<INTER>(to + m.a, to + m.b, y);
        to += kSub * p.dim;
      }
      h += kSlots;
      x += kSlots * s.x_hs;
      if (h - sub >= end) break;
      fetch<T, kRows, kSub>(x, s.x_hs, m, h, end, raw);
    }
  }
}

template <typename T, int LPR, bool INTER>
__global__ void __launch_bounds__(kWarps * 32, kResident<true>) bwd_kernel(const __grid_constant__ Params p) {
  constexpr int kRows = kRowsOf<T>, kSub = 32 / LPR, kSlots = kSub * kRows;
  __shared__ __align__(16) float sums[kWarps][kMaxDimFast];
  const Side& s = p.side[blockIdx.x >= p.side[1].first_block];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % LPR, sub = lane / LPR;
  const LaneMap m = lane_map<INTER>(l, p.dim, p.rotary);
  const uint32_t first = (blockIdx.x - s.first_block) * kWarps + warp, stride = s.blocks * kWarps;
  Lane w{}, dw{};
  if (m.active) w = weights_of<INTER>(s.w, p.w_dtype, m);
  T* const out = static_cast<T*>(s.out);
  Positions positions;
  if (s.flat) {
    const uint32_t rows = (uint32_t)p.tokens * s.heads;
    for (uint32_t item = first; item < s.items; item += stride) {
      Raw<T> rx[kRows][2], rg[kRows][2];
      uint32_t token[kRows], last = ~0u;
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const uint32_t row = item * kSlots + i * kSub + sub, t = row / (uint32_t)s.heads, h = row - t * s.heads;
        token[i] = t;
        rx[i][0].u = rx[i][1].u = rg[i][0].u = rg[i][1].u = {};
        if (row < rows && m.active) {
          const T* x = static_cast<const T*>(s.x) + t * s.x_ts + h * s.x_hs;
          const T* g = static_cast<const T*>(s.g) + t * s.g_ts + h * s.g_hs;
          rx[i][0] = load_run(x + m.a), rx[i][1] = load_run(x + m.b);
          rg[i][0] = load_run(g + m.a), rg[i][1] = load_run(g + m.b);
        }
      }
      Angles angles;
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const uint32_t row = item * kSlots + i * kSub + sub;
        const bool ok = row < rows && m.active;
        if (ok && token[i] != last) angles.load(p, positions, m, last = token[i], l);
        float fx[2 * kE], fg[2 * kE], y[2 * kE];
        unpack_lane<INTER>(rx[i], fx);
        unpack_lane<INTER>(rg[i], fg);
        bwd_row<LPR>(p, m, lane_of(fx), lane_of(fg), w, angles, ok, dw, y);
        if (ok && out) store_lane<INTER>(out + (int64_t)row * p.dim + m.a, out + (int64_t)row * p.dim + m.b, y);
      }
    }
  } else {
    for (uint32_t item = first; item < s.items; item += stride) {
      const uint32_t t = item / s.spans, chunk = (item - t * s.spans) * s.span;
      int h = (int)chunk * kSlots + sub;
      const int end = min((int)(chunk + s.span) * kSlots, s.heads);
      const T* x = static_cast<const T*>(s.x) + (int64_t)t * s.x_ts + h * s.x_hs;
      const T* g = static_cast<const T*>(s.g) + (int64_t)t * s.g_ts + h * s.g_hs;
      int64_t to = ((int64_t)t * s.heads + h) * p.dim;
      Raw<T> rx[kRows][2], rg[kRows][2];
      fetch<T, kRows, kSub>(x, s.x_hs, m, h, end, rx);
      fetch<T, kRows, kSub>(g, s.g_hs, m, h, end, rg);
      Angles angles;
      angles.load(p, positions, m, t, l);
      while (true) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          float fx[2 * kE], fg[2 * kE], y[2 * kE];
          unpack_lane<INTER>(rx[i], fx);
          unpack_lane<INTER>(rg[i], fg);
          const bool ok = h + i * kSub < end && m.active;
          bwd_row<LPR>(p, m, lane_of(fx), lane_of(fg), w, angles, ok, dw, y);
          if (ok && out) store_lane<INTER>(out + to + m.a, out + to + m.b, y);
          to += kSub * p.dim;
        }
        h += kSlots;
        x += kSlots * s.x_hs;
        g += kSlots * s.g_hs;
        if (h - sub >= end) break;
        fetch<T, kRows, kSub>(x, s.x_hs, m, h, end, rx);
        fetch<T, kRows, kSub>(g, s.g_hs, m, h, end, rg);
      }
    }
  }
  if (!p.partial) return;
  float sum[2 * kE];
  floats_of(dw, sum);
#pragma unroll
  for (int e = 0; e < 2 * kE; ++e) {
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], o);
  }
  if (lane < LPR && m.active) {
    float a[kE], b[kE];
    from_pairs<INTER>(sum, a, b);
#pragma unroll
    for (int e = 0; e < kE; ++e) sums[warp][m.a + e] = a[e], sums[warp][m.b + e] = b[e];
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.dim; d += kWarps * 32) {
    float acc = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) acc += sums[k][d];
    p.partial[(int64_t)blockIdx.x * p.dim + d] = acc;
  }
}

// ------------------------------------------------------------------ any shape
// One warp per row, element by element (head dims that are not multiples of 8 or above
// 256, rotated widths that are not, rows off the vector alignment). blockIdx.y: q or k.
template <typename T, int NU, bool BWD>
__global__ void __launch_bounds__(kWarps * 32) any_kernel(const __grid_constant__ Params p) {
  __shared__ float sums[BWD ? kWarps : 1][BWD ? kMaxDim : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Side& s = p.side[blockIdx.y];
  const int n_units = p.dim - p.rotary / 2;
  const int64_t rows = p.tokens * s.heads;
  Positions positions;
  float dw[NU][2];
#pragma unroll
  for (int j = 0; j < NU; ++j) dw[j][0] = dw[j][1] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * kWarps + warp; row < rows; row += (int64_t)gridDim.x * kWarps) {
    const int64_t t = row / s.heads;
    const int h = (int)(row - t * s.heads);
    const T* x = static_cast<const T*>(s.x) + t * s.x_ts + h * s.x_hs;
    const T* g = BWD ? static_cast<const T*>(s.g) + t * s.g_ts + h * s.g_hs : nullptr;
    const int64_t pos = positions.of(p, t);
    const bool inside = pos >= 0 && pos < p.table_rows;
    // a position outside the table turns nothing (the row is NaN through r): the table may have no rows at all
    const float* angles = p.table + (inside ? pos : 0) * p.rotary;
    auto turn = [&](float& a, float& b, int unit, float sign) {
      if (inside) rotate_pair(a, b, angles[unit], sign * angles[p.rotary / 2 + unit]);
    };
    float v[NU][2], u[BWD ? NU : 1][2], ss = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < NU; ++j) {
      const int unit = lane + 32 * j;
      v[j][0] = v[j][1] = 0.f;
      if (BWD) u[j][0] = u[j][1] = 0.f;
      if (unit >= n_units) continue;
      const Unit e = unit_of(unit, p.rotary, p.interleaved);
      v[j][0] = to_float(x[e.a]);
      if (e.b >= 0) v[j][1] = to_float(x[e.b]);
      ss = fmaf(v[j][0], v[j][0], ss);
      ss = fmaf(v[j][1], v[j][1], ss);
      if (BWD) {
        u[j][0] = to_float(g[e.a]);
        if (e.b >= 0) {
          u[j][1] = to_float(g[e.b]);
          turn(u[j][0], u[j][1], unit, -1.f);
        }
        dot = fmaf(u[j][0] * load_weight(s.w, e.a, p.w_dtype), v[j][0], dot);
        if (e.b >= 0) dot = fmaf(u[j][1] * load_weight(s.w, e.b, p.w_dtype), v[j][1], dot);
      }
    }
    ss = row_sum<32>(ss);
    const float r = inside ? rsqrtf(ss * p.inv_dim + p.eps) : nan_f32();
    const float mean = BWD ? row_sum<32>(dot) * r * p.inv_dim : 0.f;
    T* out = s.out ? static_cast<T*>(s.out) + row * p.dim : nullptr;
#pragma unroll
    for (int j = 0; j < NU; ++j) {
      const int unit = lane + 32 * j;
      if (unit >= n_units) continue;
      const Unit e = unit_of(unit, p.rotary, p.interleaved);
      const float wa = load_weight(s.w, e.a, p.w_dtype), wb = e.b >= 0 ? load_weight(s.w, e.b, p.w_dtype) : 0.f;
      float ya, yb;
      if (BWD) {
        const float ha = v[j][0] * r, hb = v[j][1] * r;
        dw[j][0] += u[j][0] * ha;
        dw[j][1] += u[j][1] * hb;
        ya = r * (u[j][0] * wa - ha * mean);
        yb = r * (u[j][1] * wb - hb * mean);
      } else {
        ya = v[j][0] * r * wa;
        yb = v[j][1] * r * wb;
        if (e.b >= 0) turn(ya, yb, unit, 1.f);
      }
      if (out) {
        out[e.a] = from_float<T>(ya);
        if (e.b >= 0) out[e.b] = from_float<T>(yb);
      }
    }
  }
  if constexpr (BWD) {
    if (!p.partial) return;
#pragma unroll
    for (int j = 0; j < NU; ++j) {
      const int unit = lane + 32 * j;
      if (unit >= n_units) continue;
      const Unit e = unit_of(unit, p.rotary, p.interleaved);
      sums[warp][e.a] = dw[j][0];
      if (e.b >= 0) sums[warp][e.b] = dw[j][1];
    }
    __syncthreads();
    for (int d = threadIdx.x; d < p.dim; d += kWarps * 32) {
      float acc = 0.f;
      for (int k = 0; k < kWarps; ++k) acc += sums[k][d];
      p.partial[((int64_t)blockIdx.x * 2 + blockIdx.y) * p.dim + d] = acc;
    }
  }
}

// ------------------------------------------------------------------ weight gradients
// 32 columns a block, its 32 warps over the blocks' partial sums; float64 from here on (a few hundred terms
// a column, free beside the reads). Row r of a side is partial[(first + r * step) * dim].
struct PartialRows {
  int first, rows, step;
};
constexpr int kDwWarps = 32;
__global__ void __launch_bounds__(kDwWarps * 32)
dw_kernel(const float* __restrict__ partial, PartialRows q_rows, PartialRows k_rows, int dim, int w_dtype,
          void* __restrict__ dwq, void* __restrict__ dwk) {
  __shared__ double sums[kDwWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = blockIdx.x * 32 + lane;
  const PartialRows at = blockIdx.y ? k_rows : q_rows;
  void* dst = blockIdx.y ? dwk : dwq;
  if (!dst) return;
  double acc = 0.0;
  if (d < dim) {
#pragma unroll 8
    for (int r = warp; r < at.rows; r += kDwWarps)
      acc += (double)partial[((int64_t)at.first + (int64_t)r * at.step) * dim + d];
  }
  sums[warp][lane] = acc;
  __syncthreads();
  if (warp != 0 || d >= dim) return;
#pragma unroll
  for (int k = 1; k < kDwWarps; ++k) acc += sums[k][lane];
  const float f = (float)acc;
  if (w_dtype == MSA_F32) reinterpret_cast<float*>(dst)[d] = f;
  else if (w_dtype == MSA_F16) reinterpret_cast<__half*>(dst)[d] = __float2half_rn(f);
  else reinterpret_cast<__nv_bfloat16*>(dst)[d] = __float2bfloat16_rn(f);
}

// ------------------------------------------------------------------ host
// Whether every row can be taken in runs of four elements.
bool runs_fit(const Params& p, int es, bool bwd) {
  if (p.dim % (2 * kE) || p.rotary % (2 * kE) || p.dim > kMaxDimFast || reinterpret_cast<uintptr_t>(p.table) % 16)
    return false;
  for (const Side& s : p.side) {
    if (!rows_aligned(s.x, s.x_ts, s.x_hs, es, kE * es) || !rows_aligned(s.out, 0, 0, es, kE * es)) return false;
    if (bwd && !rows_aligned(s.g, s.g_ts, s.g_hs, es, kE * es)) return false;
    if (p.tokens * s.heads >= (int64_t)1 << 31) return false;  // 32-bit row numbers
  }
  return true;
}

// The blocks of a launch stay on the chip; the backward's number bounds the rows of its partial sums (the
// any-shape kernel has as many for each side).
template <bool BWD>
constexpr int kMaxBlocks = 148 * kResident<BWD>;
int blocks_for(int64_t items, int most) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, (items + kWarps - 1) / kWarps));
}

// Items of both sides, and each side's share of the blocks. A flat step costs more, its angles being loaded row by
// row: in halves of another step's.
constexpr int kFlatCost = 3;
int deal(Params& p, int slots, int most) {
  int64_t steps[2], cost[2];
  for (int i = 0; i < 2; ++i) {
    Side& s = p.side[i];
    s.flat = s.heads < slots;
    s.chunks = ceil_div(s.heads, slots);
    steps[i] = s.flat ? ceil_div(p.tokens * s.heads, slots) : p.tokens * s.chunks;
    // as many steps to an item as leave every warp eight items or more
    s.span = (uint32_t)std::max<int64_t>(1, std::min<int64_t>(s.chunks, steps[i] / ((int64_t)most * kWarps * 8)));
    s.spans = ceil_div(s.chunks, s.span);
    s.items = (uint32_t)(s.flat ? steps[i] : p.tokens * s.spans);
    cost[i] = steps[i] * (s.flat ? kFlatCost : 2);
  }
  int k_blocks = (int)std::max<int64_t>(1, (most * cost[1] + (cost[0] + cost[1]) / 2) / (cost[0] + cost[1]));
  k_blocks = std::min(blocks_for(p.side[1].items, most - 1), k_blocks);
  p.side[0].first_block = 0;
  p.side[0].blocks = blocks_for(p.side[0].items, most - k_blocks);
  p.side[1].first_block = p.side[0].blocks;
  p.side[1].blocks = k_blocks;
  return p.side[0].blocks + k_blocks;
}

template <typename T, int LPR, bool BWD>
void launch_rows(Params& p, cudaStream_t st) {
  const int blocks = deal(p, 32 / LPR * kRowsOf<T>, kMaxBlocks<BWD>);
  if constexpr (BWD) {
    if (p.interleaved) bwd_kernel<T, LPR, true><<<blocks, kWarps * 32, 0, st>>>(p);
    else bwd_kernel<T, LPR, false><<<blocks, kWarps * 32, 0, st>>>(p);
  } else {
    if (p.interleaved) fwd_kernel<T, LPR, true><<<blocks, kWarps * 32, 0, st>>>(p);
    else fwd_kernel<T, LPR, false><<<blocks, kWarps * 32, 0, st>>>(p);
  }
}

template <typename T, bool BWD>
void launch_runs(Params& p, cudaStream_t st) {
  const int lanes = p.dim / (2 * kE);
  if (lanes <= 4) launch_rows<T, 4, BWD>(p, st);
  else if (lanes <= 8) launch_rows<T, 8, BWD>(p, st);
  else if (lanes <= 16) launch_rows<T, 16, BWD>(p, st);
  else launch_rows<T, 32, BWD>(p, st);
}

template <typename T>
int launch(Params p, int dtype, bool bwd, void* dwq, void* dwk, cudaStream_t st) {
  PartialRows q_rows, k_rows;
  if (runs_fit(p, elem_size(dtype), bwd)) {
    if (bwd) launch_runs<T, true>(p, st);
    else launch_runs<T, false>(p, st);
    q_rows = PartialRows{0, (int)p.side[0].blocks, 1};
    k_rows = PartialRows{(int)p.side[1].first_block, (int)p.side[1].blocks, 1};
  } else {
    const bool small = p.dim - p.rotary / 2 <= 128;
    const int blocks = blocks_for(p.tokens * std::max(p.side[0].heads, p.side[1].heads),
                                  bwd ? kMaxBlocks<true> : kMaxBlocks<false>);
    const dim3 grid(blocks, 2);
    if (bwd) {
      if (small) any_kernel<T, 4, true><<<grid, kWarps * 32, 0, st>>>(p);
      else any_kernel<T, 16, true><<<grid, kWarps * 32, 0, st>>>(p);
    } else {
      if (small) any_kernel<T, 4, false><<<grid, kWarps * 32, 0, st>>>(p);
      else any_kernel<T, 16, false><<<grid, kWarps * 32, 0, st>>>(p);
    }
    q_rows = PartialRows{0, blocks, 2};
    k_rows = PartialRows{1, blocks, 2};
  }
  count_launches(1);
  if (int e = launch_status("qk_norm_rope")) return e;
  if (bwd && p.partial) {
    dw_kernel<<<dim3(ceil_div(p.dim, 32), 2), kDwWarps * 32, 0, st>>>(p.partial, q_rows, k_rows, p.dim, p.w_dtype,
                                                                      dwq, dwk);
    count_launches(1);
    return launch_status("qk_norm_rope dw");
  }
  return MSA_OK;
}

int check(const char* what, int dtype, int w_dtype, int64_t tokens, int32_t q_heads, int32_t k_heads, int32_t dim,
          int32_t rotary, int64_t table_rows, const int32_t* positions, const int32_t* cu, int32_t nseq, double eps) {
  MSA_CHECK_ARG(valid_dtype(dtype) && (w_dtype == dtype || w_dtype == MSA_F32), "%s: bad dtype", what);
  MSA_CHECK_ARG(tokens >= 0 && q_heads >= 1 && k_heads >= 1, "%s: bad sizes", what);
  MSA_CHECK_ARG(dim >= 1 && dim <= kMaxDim, "%s: head_dim must be in [1, %d]", what, kMaxDim);
  MSA_CHECK_ARG(rotary >= 0 && rotary % 2 == 0 && rotary <= dim && table_rows >= 0,
                "%s: rotary_dim must be even and at most head_dim", what);
  MSA_CHECK_ARG((positions != nullptr) != (cu != nullptr) || tokens == 0,
                "%s: give positions or cu_seqlens", what);
  MSA_CHECK_ARG(positions || tokens == 0 || nseq >= 1, "%s: cu_seqlens needs a sequence", what);
  MSA_CHECK_ARG(eps >= 0, "%s: eps must not be negative", what);
  return MSA_OK;
}

}  // namespace
}  // namespace msa

using namespace msa;

extern "C" int msa_qk_norm_rope_fwd(const void* q, const void* k, int dtype, const void* q_weight,
                                    const void* k_weight, int weight_dtype, const float* rope_table,
                                    int64_t table_rows, int32_t rotary_dim, int interleaved,
                                    const int32_t* positions, const int32_t* cu_seqlens, int32_t nseq,
                                    int64_t total_tokens, int32_t q_heads, int32_t k_heads, int32_t head_dim,
                                    int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                                    int64_t k_head_stride, double eps, void* q_out, void* k_out, void* stream) {
  if (int e = check("msa_qk_norm_rope_fwd", dtype, weight_dtype, total_tokens, q_heads, k_heads, head_dim, rotary_dim,
                    table_rows, positions, cu_seqlens, nseq, eps))
    return e;
  if (total_tokens == 0) return MSA_OK;
  Params p{};
  p.side[0] = Side{q, q_weight, nullptr, q_out, q_token_stride, q_head_stride, 0, 0, q_heads};
  p.side[1] = Side{k, k_weight, nullptr, k_out, k_token_stride, k_head_stride, 0, 0, k_heads};
  p.table = rope_table, p.table_rows = table_rows, p.positions = positions, p.cu = cu_seqlens, p.nseq = nseq;
  p.tokens = total_tokens, p.dim = head_dim, p.rotary = rotary_dim, p.w_dtype = weight_dtype;
  p.eps = (float)eps, p.inv_dim = 1.f / head_dim, p.interleaved = interleaved != 0;
  cudaStream_t st = as_stream(stream);
  if (dtype == MSA_BF16) return launch<__nv_bfloat16>(p, dtype, false, nullptr, nullptr, st);
  if (dtype == MSA_F16) return launch<__half>(p, dtype, false, nullptr, nullptr, st);
  return launch<float>(p, dtype, false, nullptr, nullptr, st);
}

extern "C" size_t msa_qk_norm_rope_bwd_workspace_size(int32_t head_dim) {
  return sizeof(float) * 2 * (size_t)kMaxBlocks<true> * head_dim;
}

extern "C" int msa_qk_norm_rope_bwd(const void* q, const void* k, const void* grad_q, const void* grad_k, int dtype,
                                    const void* q_weight, const void* k_weight, int weight_dtype,
                                    const float* rope_table, int64_t table_rows, int32_t rotary_dim, int interleaved,
                                    const int32_t* positions, const int32_t* cu_seqlens, int32_t nseq,
                                    int64_t total_tokens, int32_t q_heads, int32_t k_heads, int32_t head_dim,
                                    int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                                    int64_t k_head_stride, int64_t gq_token_stride, int64_t gq_head_stride,
                                    int64_t gk_token_stride, int64_t gk_head_stride, double eps, void* dq, void* dk,
                                    void* dq_weight, void* dk_weight, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  if (int e = check("msa_qk_norm_rope_bwd", dtype, weight_dtype, total_tokens, q_heads, k_heads, head_dim, rotary_dim,
                    table_rows, positions, cu_seqlens, nseq, eps))
    return e;
  const bool weights = dq_weight || dk_weight;
  MSA_CHECK_ARG(!weights || workspace_bytes >= msa_qk_norm_rope_bwd_workspace_size(head_dim),
                "msa_qk_norm_rope_bwd: workspace too small");
  cudaStream_t st = as_stream(stream);
  if (total_tokens == 0) {  // no rows: the weights' gradients are zero
    const size_t bytes = (size_t)head_dim * elem_size(weight_dtype);
    if (dq_weight) MSA_CUDA_RETURN(cudaMemsetAsync(dq_weight, 0, bytes, st));
    if (dk_weight) MSA_CUDA_RETURN(cudaMemsetAsync(dk_weight, 0, bytes, st));
    return MSA_OK;
  }
  Params p{};
  p.side[0] = Side{q, q_weight, grad_q, dq, q_token_stride, q_head_stride, gq_token_stride, gq_head_stride, q_heads};
  p.side[1] = Side{k, k_weight, grad_k, dk, k_token_stride, k_head_stride, gk_token_stride, gk_head_stride, k_heads};
  p.table = rope_table, p.table_rows = table_rows, p.positions = positions, p.cu = cu_seqlens, p.nseq = nseq;
  p.partial = weights ? static_cast<float*>(workspace) : nullptr;
  p.tokens = total_tokens, p.dim = head_dim, p.rotary = rotary_dim, p.w_dtype = weight_dtype;
  p.eps = (float)eps, p.inv_dim = 1.f / head_dim, p.interleaved = interleaved != 0;
  if (dtype == MSA_BF16) return launch<__nv_bfloat16>(p, dtype, true, dq_weight, dk_weight, st);
  if (dtype == MSA_F16) return launch<__half>(p, dtype, true, dq_weight, dk_weight, st);
  return launch<float>(p, dtype, true, dq_weight, dk_weight, st);
}
