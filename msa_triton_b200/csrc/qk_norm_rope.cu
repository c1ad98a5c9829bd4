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
// an element) instead of storing it. q and k go through one launch. The weights' gradients
// are summed in registers by persistent warps, then over a block's warps and the blocks in a
// fixed order (no atomics, the same bits every run).
#include <algorithm>

#include "rope_common.cuh"

namespace msa {
namespace {

using namespace rope;

constexpr int kWarps = 8;
constexpr int kRowsPerLane = 4;   // rows a lane loads before it uses the first (forward)
constexpr int kRowsPerLaneB = 2;  // (backward: two tensors a row)
constexpr int kMaxDimFast = 256;
constexpr int kMaxDim = 512;

// One of q and k.
struct Side {
  const void* x;
  const void* w;
  const void* g;  // backward: gradient of the output
  void* out;      // forward: y; backward: dx (may be null)
  int64_t x_ts, x_hs, g_ts, g_hs;  // strides in elements
  int heads;
};

struct Params {
  Side side[2];
  const float* table;
  const int32_t* positions;  // or null: from cu
  const int32_t* cu;
  float* partial;  // backward: [gridDim.x][2][dim], or null
  int64_t table_rows, tokens;
  int nseq, dim, rotary, w_dtype;
  uint32_t units, chunks, q_chunks;
  float eps, inv_dim;
  bool interleaved;
};

__device__ __forceinline__ int64_t position_of(const Params& p, int64_t t) {
  if (p.positions) return p.positions[t];
  return t - p.cu[find_sequence(p.cu, p.nseq, t)];
}

__device__ __forceinline__ float load_weight(const void* w, int i, int dtype) {
  if (dtype == MSA_F32) return reinterpret_cast<const float*>(w)[i];
  if (dtype == MSA_F16) return __half2float(reinterpret_cast<const __half*>(w)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[i]);
}

template <bool INTER>
__device__ __forceinline__ void load_weights(const void* w, int dtype, const LaneMap& m, float (&v)[8]) {
  float a[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = load_weight(w, m.a + i, dtype), b[i] = load_weight(w, m.b + i, dtype);
  to_pairs<INTER>(a, b, v);
}

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// ------------------------------------------------------------------ forward
// A warp takes 32 / LPR * kRowsPerLane heads of one token (q's or k's); the angles are
// loaded once for them.
template <typename T, int LPR, bool INTER>
__global__ void __launch_bounds__(kWarps * 32) fwd_kernel(const __grid_constant__ Params p) {
  constexpr int kSub = 32 / LPR;
  const uint32_t unit = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (unit >= p.units) return;
  const uint32_t t = unit / p.chunks;
  uint32_t chunk = unit - t * p.chunks;
  const int lane = threadIdx.x & 31, l = lane % LPR;
  const bool is_k = chunk >= p.q_chunks;
  if (is_k) chunk -= p.q_chunks;
  const Side& s = p.side[is_k];
  const LaneMap m = lane_map<INTER>(l, p.dim, p.rotary);
  const int h0 = chunk * (kSub * kRowsPerLane) + lane / LPR;
  const T* x = static_cast<const T*>(s.x) + (int64_t)t * s.x_ts;
  Raw4<T> raw[kRowsPerLane][2];
#pragma unroll
  for (int i = 0; i < kRowsPerLane; ++i) {
    const int h = h0 + i * kSub;
    if (h < s.heads && m.active) {
      raw[i][0] = load4(x + h * s.x_hs + m.a);
      raw[i][1] = load4(x + h * s.x_hs + m.b);
    } else {
      raw[i][0].u = raw[i][1].u = {};
    }
  }
  const int64_t pos = position_of(p, t);
  const bool inside = pos >= 0 && pos < p.table_rows;
  float c[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f}, w[8];
  if (inside && m.rotated) load_angles(p.table + pos * p.rotary, p.rotary, l, c, sn);
  if (m.active) load_weights<INTER>(s.w, p.w_dtype, m, w);
  T* out = static_cast<T*>(s.out) + (int64_t)t * s.heads * p.dim;
#pragma unroll
  for (int i = 0; i < kRowsPerLane; ++i) {
    float a[4], b[4], v[8], ss = 0.f;
    unpack4(raw[i][0], a);
    unpack4(raw[i][1], b);
    to_pairs<INTER>(a, b, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
    ss = row_sum<LPR>(ss);
    const float r = inside ? rsqrtf(ss * p.inv_dim + p.eps) : nan_f32();
    const int h = h0 + i * kSub;
    if (h < s.heads && m.active) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * r * w[e];
      if (m.rotated) rotate8(v, c, sn);
      store8<INTER>(out + (int64_t)h * p.dim, m, v);
    }
  }
}

// ------------------------------------------------------------------ backward
template <typename T, int LPR, bool INTER>
__global__ void __launch_bounds__(kWarps * 32) bwd_kernel(const __grid_constant__ Params p) {
  constexpr int kSub = 32 / LPR;
  __shared__ __align__(16) float sums[kWarps][kMaxDimFast];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % LPR;
  const LaneMap m = lane_map<INTER>(l, p.dim, p.rotary);
  float dw[2][8], w[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[0][e] = dw[1][e] = 0.f, w[0][e] = w[1][e] = 0.f;
  if (m.active) {
    load_weights<INTER>(p.side[0].w, p.w_dtype, m, w[0]);
    load_weights<INTER>(p.side[1].w, p.w_dtype, m, w[1]);
  }
  for (uint32_t unit = blockIdx.x * kWarps + warp; unit < p.units; unit += gridDim.x * kWarps) {
    const uint32_t t = unit / p.chunks;
    uint32_t chunk = unit - t * p.chunks;
    const bool is_k = chunk >= p.q_chunks;
    if (is_k) chunk -= p.q_chunks;
    const Side& s = p.side[is_k];
    const int h0 = chunk * (kSub * kRowsPerLaneB) + lane / LPR;
    const T* x = static_cast<const T*>(s.x) + (int64_t)t * s.x_ts;
    const T* g = static_cast<const T*>(s.g) + (int64_t)t * s.g_ts;
    Raw4<T> rx[kRowsPerLaneB][2], rg[kRowsPerLaneB][2];
#pragma unroll
    for (int i = 0; i < kRowsPerLaneB; ++i) {
      const int h = h0 + i * kSub;
      if (h < s.heads && m.active) {
        rx[i][0] = load4(x + h * s.x_hs + m.a);
        rx[i][1] = load4(x + h * s.x_hs + m.b);
        rg[i][0] = load4(g + h * s.g_hs + m.a);
        rg[i][1] = load4(g + h * s.g_hs + m.b);
      } else {
        rx[i][0].u = rx[i][1].u = {};
        rg[i][0].u = rg[i][1].u = {};
      }
    }
    const int64_t pos = position_of(p, t);
    const bool inside = pos >= 0 && pos < p.table_rows;
    float c[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
    if (inside && m.rotated) load_angles(p.table + pos * p.rotary, p.rotary, l, c, sn);
#pragma unroll
    for (int e = 0; e < 4; ++e) sn[e] = -sn[e];  // the transposed rotation
#pragma unroll
    for (int i = 0; i < kRowsPerLaneB; ++i) {
      float a[4], b[4], v[8], u[8], ss = 0.f, dot = 0.f;
      unpack4(rx[i][0], a);
      unpack4(rx[i][1], b);
      to_pairs<INTER>(a, b, v);
      unpack4(rg[i][0], a);
      unpack4(rg[i][1], b);
      to_pairs<INTER>(a, b, u);
      if (m.rotated) rotate8(u, c, sn);
      // both sums in one round of shuffles: mean(u * x') = r mean(u * x)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss = fmaf(v[e], v[e], ss);
        dot = fmaf(u[e] * (is_k ? w[1][e] : w[0][e]), v[e], dot);
      }
      ss = row_sum<LPR>(ss);
      dot = row_sum<LPR>(dot);
      const int h = h0 + i * kSub;
      const bool mine = h < s.heads && m.active;
      const float r = inside ? rsqrtf(ss * p.inv_dim + p.eps) : nan_f32();
      const float mean = dot * r * p.inv_dim;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float hat = v[e] * r;
        // rows past the last head count nothing (their r is eps^-1/2, or NaN)
        const float part = mine ? u[e] * hat : 0.f;
        if (is_k) dw[1][e] += part; else dw[0][e] += part;
        v[e] = r * (u[e] * (is_k ? w[1][e] : w[0][e]) - hat * mean);
      }
      if (mine && s.out) store8<INTER>(static_cast<T*>(s.out) + ((int64_t)t * s.heads + h) * p.dim, m, v);
    }
  }
  if (!p.partial) return;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1) dw[side][e] += __shfl_xor_sync(0xffffffffu, dw[side][e], o);
    }
    if (lane < LPR && m.active) store8<INTER>(&sums[warp][0], m, dw[side]);
    __syncthreads();
    for (int d = threadIdx.x; d < p.dim; d += kWarps * 32) {
      float acc = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) acc += sums[k][d];
      p.partial[((int64_t)blockIdx.x * 2 + side) * p.dim + d] = acc;
    }
    __syncthreads();
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
  float dw[NU][2];
#pragma unroll
  for (int j = 0; j < NU; ++j) dw[j][0] = dw[j][1] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * kWarps + warp; row < rows; row += (int64_t)gridDim.x * kWarps) {
    const int64_t t = row / s.heads;
    const int h = (int)(row - t * s.heads);
    const T* x = static_cast<const T*>(s.x) + t * s.x_ts + h * s.x_hs;
    const T* g = BWD ? static_cast<const T*>(s.g) + t * s.g_ts + h * s.g_hs : nullptr;
    const int64_t pos = position_of(p, t);
    const bool inside = pos >= 0 && pos < p.table_rows;
    const float* angles = p.table + (inside ? pos : 0) * p.rotary;
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
          rotate_pair(u[j][0], u[j][1], angles[unit], -angles[p.rotary / 2 + unit]);
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
        if (e.b >= 0) rotate_pair(ya, yb, angles[unit], angles[p.rotary / 2 + unit]);
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
// 32 columns a block, its 8 warps over the blocks' partial sums; float64 from here on
// (a few hundred terms a column, free beside the reads).
__global__ void __launch_bounds__(kWarps * 32)
dw_kernel(const float* __restrict__ partial, int blocks, int dim, int w_dtype, void* __restrict__ dwq,
          void* __restrict__ dwk) {
  __shared__ double sums[kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int d = blockIdx.x * 32 + lane, side = blockIdx.y;
  void* dst = side ? dwk : dwq;
  if (!dst) return;
  double acc = 0.0;
  if (d < dim)
    for (int b = warp; b < blocks; b += kWarps) acc += (double)partial[((int64_t)b * 2 + side) * dim + d];
  sums[warp][lane] = acc;
  __syncthreads();
  if (warp != 0 || d >= dim) return;
  for (int k = 1; k < kWarps; ++k) acc += sums[k][lane];
  const float f = (float)acc;
  if (w_dtype == MSA_F32) reinterpret_cast<float*>(dst)[d] = f;
  else if (w_dtype == MSA_F16) reinterpret_cast<__half*>(dst)[d] = __float2half_rn(f);
  else reinterpret_cast<__nv_bfloat16*>(dst)[d] = __float2bfloat16_rn(f);
}

// ------------------------------------------------------------------ host
int lanes_per_row(int dim) { return dim <= 32 ? 4 : dim <= 64 ? 8 : dim <= 128 ? 16 : 32; }

bool fast_shape(const Params& p, int dtype, bool bwd) {
  const int es = elem_size(dtype);
  if (p.dim % 8 || p.rotary % 8 || p.dim > kMaxDimFast || reinterpret_cast<uintptr_t>(p.table) % 16) return false;
  for (const Side& s : p.side) {
    if (!rows_aligned(s.x, s.x_ts, s.x_hs, es) || !rows_aligned(s.out, 0, 0, es)) return false;
    if (bwd && !rows_aligned(s.g, s.g_ts, s.g_hs, es)) return false;
  }
  return true;
}

// Blocks of the backward (and rows of its partial sums): enough for the chip, no more
// than there is work.
constexpr int kBwdBlocks = 148 * 6;
int bwd_blocks(int64_t units) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(kBwdBlocks, (units + kWarps - 1) / kWarps));
}

template <typename T, int LPR>
void launch_fast(const Params& p, bool bwd, int blocks, cudaStream_t st) {
  if (bwd) {
    if (p.interleaved) bwd_kernel<T, LPR, true><<<blocks, kWarps * 32, 0, st>>>(p);
    else bwd_kernel<T, LPR, false><<<blocks, kWarps * 32, 0, st>>>(p);
  } else {
    if (p.interleaved) fwd_kernel<T, LPR, true><<<blocks, kWarps * 32, 0, st>>>(p);
    else fwd_kernel<T, LPR, false><<<blocks, kWarps * 32, 0, st>>>(p);
  }
}

template <typename T>
int launch(Params p, int dtype, bool bwd, void* dwq, void* dwk, cudaStream_t st) {
  int blocks;
  if (fast_shape(p, dtype, bwd)) {
    const int lpr = lanes_per_row(p.dim);
    const int rows = 32 / lpr * (bwd ? kRowsPerLaneB : kRowsPerLane);
    p.q_chunks = ceil_div(p.side[0].heads, rows);
    p.chunks = p.q_chunks + ceil_div(p.side[1].heads, rows);
    const int64_t units = p.tokens * p.chunks;
    MSA_CHECK_ARG(units < (int64_t)1 << 31, "msa_qk_norm_rope: too many tokens * heads");
    p.units = (uint32_t)units;
    blocks = bwd ? bwd_blocks(units) : ceil_div(units, kWarps);
    switch (lpr) {
      case 4: launch_fast<T, 4>(p, bwd, blocks, st); break;
      case 8: launch_fast<T, 8>(p, bwd, blocks, st); break;
      case 16: launch_fast<T, 16>(p, bwd, blocks, st); break;
      default: launch_fast<T, 32>(p, bwd, blocks, st); break;
    }
  } else {
    const bool small = p.dim - p.rotary / 2 <= 128;
    blocks = bwd_blocks(p.tokens * std::max(p.side[0].heads, p.side[1].heads));
    const dim3 grid(blocks, 2);
    if (bwd) {
      if (small) any_kernel<T, 4, true><<<grid, kWarps * 32, 0, st>>>(p);
      else any_kernel<T, 16, true><<<grid, kWarps * 32, 0, st>>>(p);
    } else {
      if (small) any_kernel<T, 4, false><<<grid, kWarps * 32, 0, st>>>(p);
      else any_kernel<T, 16, false><<<grid, kWarps * 32, 0, st>>>(p);
    }
  }
  count_launches(1);
  if (int e = launch_status("qk_norm_rope")) return e;
  if (bwd && p.partial) {
    dw_kernel<<<dim3(ceil_div(p.dim, 32), 2), kWarps * 32, 0, st>>>(p.partial, blocks, p.dim, p.w_dtype, dwq, dwk);
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
  return sizeof(float) * 2 * (size_t)kBwdBlocks * head_dim;
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
