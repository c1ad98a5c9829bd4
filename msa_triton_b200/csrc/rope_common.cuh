// Element access and position rotation shared by the per-head norm / rotation
// kernels and the cache append.
//
// A head row of D elements is spread over D / 8 lanes, two runs of kE = 4 consecutive elements a lane, chosen
// so that both elements of every rotated pair sit in one lane and no shuffle is needed: with half-split
// pairs (i, i + R/2) lane l holds the runs at 4 l and R/2 + 4 l; lanes past the rotated R elements hold theirs
// the same way. With adjacent pairs (2i, 2i + 1) lane l holds 8 elements in a row. Pair i of a lane has angle
// index 4 l + i either way. (Runs of eight 16-bit elements halve the instructions an element but double the
// registers of a row: fewer rows in flight, and 224 instead of 210 us at 32768 tokens of 72 heads of 128.)
#pragma once

#include "common.cuh"

namespace msa {
namespace rope {

constexpr int kE = 4;

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

// ------------------------------------------------------------------ runs of four elements as they are stored
template <typename T>
struct Raw {
  uint2 u;
};
template <>
struct Raw<float> {
  uint4 u;
};

template <typename T>
__device__ __forceinline__ Raw<T> load_run(const T* p) {
  Raw<T> r;
  r.u = __ldcs(reinterpret_cast<const decltype(r.u)*>(p));  // streamed: every row is read once per pass
  return r;
}

// The same for rows that are read again soon.
template <typename T>
__device__ __forceinline__ Raw<T> load_run_again(const T* p) {
  Raw<T> r;
  r.u = __ldg(reinterpret_cast<const decltype(r.u)*>(p));
  return r;
}

__device__ __forceinline__ void unpack_word(uint32_t w, __half, float& a, float& b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  a = f.x, b = f.y;
}
__device__ __forceinline__ void unpack_word(uint32_t w, __nv_bfloat16, float& a, float& b) {
  a = __uint_as_float(w << 16), b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack_word(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_word(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void unpack_run(const Raw<float>& r, float (&f)[4]) {
  f[0] = __uint_as_float(r.u.x), f[1] = __uint_as_float(r.u.y), f[2] = __uint_as_float(r.u.z),
  f[3] = __uint_as_float(r.u.w);
}
template <typename T>
__device__ __forceinline__ void unpack_run(const Raw<T>& r, float (&f)[4]) {
  unpack_word(r.u.x, T(), f[0], f[1]);
  unpack_word(r.u.y, T(), f[2], f[3]);
}

__device__ __forceinline__ void store_run(float* p, const float (&f)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
}
template <typename T>
__device__ __forceinline__ void store_run(T* p, const float (&f)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_word(f[0], f[1], T()), pack_word(f[2], f[3], T()));
}
// Where lane l of a row finds its elements.
struct LaneMap {
  int a, b;      // element offsets of its two runs
  bool active;   // the lane holds elements at all
  bool rotated;  // they form rotated pairs (angle indices 4 l .. 4 l + 3)
};

template <bool INTER>
__device__ __forceinline__ LaneMap lane_map(int l, int dim, int rotary) {
  LaneMap m;
  m.active = l * 2 * kE < dim;
  m.rotated = l * 2 * kE < rotary;
  if (INTER) {
    m.a = 2 * kE * l;
    m.b = m.a + kE;
  } else if (m.rotated) {
    m.a = kE * l;
    m.b = rotary / 2 + kE * l;
  } else {
    m.a = rotary + kE * (l - rotary / (2 * kE));
    m.b = m.a + (dim - rotary) / 2;
  }
  return m;
}

// The lane's elements in pair order: pair i is (v[i], v[i + kE]); and back.
template <bool INTER>
__device__ __forceinline__ void to_pairs(const float (&a)[kE], const float (&b)[kE], float (&v)[2 * kE]) {
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    if (INTER) {
      v[i] = 2 * i < kE ? a[2 * i % kE] : b[2 * i % kE];
      v[i + kE] = 2 * i < kE ? a[2 * i % kE + 1] : b[2 * i % kE + 1];
    } else {
      v[i] = a[i], v[i + kE] = b[i];
    }
  }
}
template <bool INTER>
__device__ __forceinline__ void from_pairs(const float (&v)[2 * kE], float (&a)[kE], float (&b)[kE]) {
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    if (INTER) {
      (2 * i < kE ? a[2 * i % kE] : b[2 * i % kE]) = v[i];
      (2 * i < kE ? a[2 * i % kE + 1] : b[2 * i % kE + 1]) = v[i + kE];
    } else {
      a[i] = v[i], b[i] = v[i + kE];
    }
  }
}

template <bool INTER, typename T>
__device__ __forceinline__ void unpack_lane(const Raw<T> (&raw)[2], float (&v)[2 * kE]) {
  float a[kE], b[kE];
  unpack_run(raw[0], a);
  unpack_run(raw[1], b);
  to_pairs<INTER>(a, b, v);
}

template <bool INTER, typename T>
__device__ __forceinline__ void store_lane(T* a_at, T* b_at, const float (&v)[2 * kE]) {
  float a[kE], b[kE];
  from_pairs<INTER>(v, a, b);
  store_run(a_at, a);
  store_run(b_at, b);
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

// The lane's kE (cos, sin) of a table row (cos half, then sin half; 16-byte aligned).
__device__ __forceinline__ void load_angles(const float* table_row, int rotary, int l, float (&c)[kE], float (&s)[kE]) {
#pragma unroll
  for (int i = 0; i < kE / 4; ++i) {
    const float4 cc = __ldg(reinterpret_cast<const float4*>(table_row) + l * (kE / 4) + i);
    const float4 ss = __ldg(reinterpret_cast<const float4*>(table_row + rotary / 2) + l * (kE / 4) + i);
    c[4 * i] = cc.x, c[4 * i + 1] = cc.y, c[4 * i + 2] = cc.z, c[4 * i + 3] = cc.w;
    s[4 * i] = ss.x, s[4 * i + 1] = ss.y, s[4 * i + 2] = ss.z, s[4 * i + 3] = ss.w;
  }
}

__device__ __forceinline__ void rotate_lane(float (&v)[2 * kE], const float (&c)[kE], const float (&s)[kE]) {
#pragma unroll
  for (int i = 0; i < kE; ++i) rotate_pair(v[i], v[i + kE], c[i], s[i]);
}

__device__ __forceinline__ float nan_f32() { return __int_as_float(0x7fc00000); }

// ------------------------------------------------------------------ two floats to an instruction
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(F2 x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 twice(float a) { return pack2(a, a); }

// The 2 kE values of a lane, kE pairs of registers: v[0 .. kE/2-1] the pairs' first elements, the rest the second.
struct Lane {
  F2 v[kE];
};
__device__ __forceinline__ Lane lane_of(const float (&f)[2 * kE]) {
  Lane r;
#pragma unroll
  for (int i = 0; i < kE; ++i) r.v[i] = pack2(f[2 * i], f[2 * i + 1]);
  return r;
}
__device__ __forceinline__ void floats_of(const Lane& x, float (&f)[2 * kE]) {
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    const float2 t = unpack2(x.v[i]);
    f[2 * i] = t.x, f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ float dot_of(const Lane& x, const Lane& y) {
  F2 acc = mul2(x.v[0], y.v[0]);
#pragma unroll
  for (int i = 1; i < kE; ++i) acc = fma2(x.v[i], y.v[i], acc);
  const float2 t = unpack2(acc);
  return t.x + t.y;
}

// A lane's angles, ready for rotate_exact.
struct Angle2 {
  F2 c[kE / 2], s[kE / 2];
  __device__ __forceinline__ void load(const float* cos4, const float* sin4) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(cos4)), y = __ldg(reinterpret_cast<const float4*>(sin4));
    c[0] = pack2(x.x, x.y), c[1] = pack2(x.z, x.w);
    s[0] = pack2(y.x, y.y), s[1] = pack2(y.z, y.w);
  }
};
// rotate_pair with its roundings, the products of two pairs to an instruction. The sums are single instructions:
// a two-float sum of two-float products came out as a fused one although both name their rounding (a few in a
// million codes differed from rotate_pair's).
__device__ __forceinline__ void rotate_exact(Lane& x, const Angle2& t) {
#pragma unroll
  for (int i = 0; i < kE / 2; ++i) {
    const F2 a = x.v[i], b = x.v[kE / 2 + i];
    const float2 ac = unpack2(mul2(a, t.c[i])), bs = unpack2(mul2(b, t.s[i]));
    const float2 bc = unpack2(mul2(b, t.c[i])), as = unpack2(mul2(a, t.s[i]));
    x.v[i] = pack2(__fsub_rn(ac.x, bs.x), __fsub_rn(ac.y, bs.y));
    x.v[kE / 2 + i] = pack2(__fadd_rn(bc.x, as.x), __fadd_rn(bc.y, as.y));
  }
}

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

// Host: whether rows of this tensor can be read `bytes` at a time.
inline bool rows_aligned(const void* p, int64_t stride0, int64_t stride1, int elem_bytes, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride0 * elem_bytes % bytes == 0 &&
         stride1 * elem_bytes % bytes == 0;
}

inline int elem_size(int dtype) { return dtype == MSA_F32 ? 4 : 2; }

}  // namespace rope
}  // namespace msa
