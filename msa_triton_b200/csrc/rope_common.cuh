// Element access and position rotation shared by the per-head norm / rotation
// kernels and the cache append.
//
// A head row of D elements (D a multiple of 8) is spread over D / 8 lanes, eight
// elements a lane, chosen so that both elements of every rotated pair sit in one
// lane and no shuffle is needed: with half-split pairs (i, i + R/2) lane l holds
// elements 4l..4l+3 and R/2+4l..R/2+4l+3; with adjacent pairs (2i, 2i + 1) it holds
// 8l..8l+7. Lanes past the rotated R elements hold eight elements in a row. Both
// are two four-element loads (8 bytes at 16 bits, 16 bytes at 32), and pair i of the
// lane is (v[i], v[i + 4]) with angle index 4l + i either way.
#pragma once

#include "common.cuh"

namespace msa {
namespace rope {

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Four elements as they are stored (raw) and as floats.
template <typename T>
struct Raw4 {
  uint2 u;
};
template <>
struct Raw4<float> {
  uint4 u;
};

template <typename T>
__device__ __forceinline__ Raw4<T> load4(const T* p) {
  Raw4<T> r;
  r.u = __ldcs(reinterpret_cast<const decltype(r.u)*>(p));  // streamed: every row is read once per pass
  return r;
}

__device__ __forceinline__ void unpack4(const Raw4<float>& r, float (&f)[4]) {
  f[0] = __uint_as_float(r.u.x), f[1] = __uint_as_float(r.u.y), f[2] = __uint_as_float(r.u.z),
  f[3] = __uint_as_float(r.u.w);
}
__device__ __forceinline__ void unpack4(const Raw4<__half>& r, float (&f)[4]) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&r.u.y));
  f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}
__device__ __forceinline__ void unpack4(const Raw4<__nv_bfloat16>& r, float (&f)[4]) {
  f[0] = __uint_as_float(r.u.x << 16), f[1] = __uint_as_float(r.u.x & 0xffff0000u);
  f[2] = __uint_as_float(r.u.y << 16), f[3] = __uint_as_float(r.u.y & 0xffff0000u);
}

__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
__device__ __forceinline__ void store4(__half* p, float a, float b, float c, float d) {
  const __half2 x = __floats2half2_rn(a, b), y = __floats2half2_rn(c, d);
  *reinterpret_cast<uint2*>(p) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, float a, float b, float c, float d) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
  *reinterpret_cast<uint2*>(p) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// Where lane l of a row finds its elements.
struct LaneMap {
  int a, b;      // element offsets of its two four-element runs
  bool active;   // the lane holds elements at all
  bool rotated;  // they form rotated pairs (angle indices 4l .. 4l+3)
};

template <bool INTER>
__device__ __forceinline__ LaneMap lane_map(int l, int dim, int rotary) {
  LaneMap m;
  m.active = l * 8 < dim;
  m.rotated = l * 8 < rotary;
  if (!INTER && m.rotated) {
    m.a = 4 * l;
    m.b = rotary / 2 + 4 * l;
  } else {
    m.a = 8 * l;
    m.b = 8 * l + 4;
  }
  return m;
}

// The lane's eight elements in pair order: pair i is (v[i], v[i + 4]).
template <bool INTER>
__device__ __forceinline__ void to_pairs(const float (&a)[4], const float (&b)[4], float (&v)[8]) {
  if (INTER) {
    v[0] = a[0], v[4] = a[1], v[1] = a[2], v[5] = a[3];
    v[2] = b[0], v[6] = b[1], v[3] = b[2], v[7] = b[3];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[i + 4] = b[i];
  }
}

template <bool INTER, typename T>
__device__ __forceinline__ void load8(const T* row, const LaneMap& m, float (&v)[8]) {
  float a[4], b[4];
  unpack4(load4(row + m.a), a);
  unpack4(load4(row + m.b), b);
  to_pairs<INTER>(a, b, v);
}

template <bool INTER, typename T>
__device__ __forceinline__ void store8(T* row, const LaneMap& m, const float (&v)[8]) {
  if (INTER) {
    store4(row + m.a, v[0], v[4], v[1], v[5]);
    store4(row + m.b, v[2], v[6], v[3], v[7]);
  } else {
    store4(row + m.a, v[0], v[1], v[2], v[3]);
    store4(row + m.b, v[4], v[5], v[6], v[7]);
  }
}

// Rotation of one pair. Each product and sum is rounded by itself (no fused
// multiply-add), so a rotated value has the same bits wherever it is computed:
// the 8-bit append takes a page's maximum in one pass and its codes in another.
__device__ __forceinline__ void rotate_pair(float& x, float& y, float c, float s) {
  const float a = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
  const float b = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
  x = a;
  y = b;
}

// The lane's four (cos, sin) of a table row (cos half, then sin half; 16-byte aligned).
__device__ __forceinline__ void load_angles(const float* table_row, int rotary, int l, float (&c)[4], float (&s)[4]) {
  const float4 cc = __ldg(reinterpret_cast<const float4*>(table_row) + l);
  const float4 ss = __ldg(reinterpret_cast<const float4*>(table_row + rotary / 2) + l);
  c[0] = cc.x, c[1] = cc.y, c[2] = cc.z, c[3] = cc.w;
  s[0] = ss.x, s[1] = ss.y, s[2] = ss.z, s[3] = ss.w;
}

__device__ __forceinline__ void rotate8(float (&v)[8], const float (&c)[4], const float (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) rotate_pair(v[i], v[i + 4], c[i], s[i]);
}

__device__ __forceinline__ float nan_f32() { return __int_as_float(0x7fc00000); }

// ------------------------------------------------------------------ shapes the lane layout does not cover
// Unit u of a row: the pair u of the rotated elements, or one element behind them.
struct Unit {
  int a, b;  // element offsets; b < 0: a single, unrotated element
};
__device__ __forceinline__ Unit unit_of(int u, int rotary, bool interleaved) {
  const int half = rotary / 2;
  if (u >= half) return Unit{rotary + u - half, -1};
  return interleaved ? Unit{2 * u, 2 * u + 1} : Unit{u, u + half};
}

// Host: whether rows of this tensor can be read four elements at a time.
inline bool rows_aligned(const void* p, int64_t stride0, int64_t stride1, int elem_bytes) {
  return reinterpret_cast<uintptr_t>(p) % (4 * elem_bytes) == 0 && stride0 % 4 == 0 && stride1 % 4 == 0;
}

inline int elem_size(int dtype) { return dtype == MSA_F32 ? 4 : 2; }

}  // namespace rope
}  // namespace msa
