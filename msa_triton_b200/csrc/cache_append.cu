// New keys and values into a paged cache, the keys rotated by their positions on the way:
// the step before decode.cu's kernels read the cache (layout: a block table maps each
// request's logical pages to physical pages, as there).
//
// Request b's new tokens are rows cu[b] .. cu[b+1]-1 of k and v (without cu: row b) and take the
// last positions of its seq_lens[b] tokens. Token at position p goes to row p % S of physical page
// block_table[b][p / S]. Rows behind the last request, positions below 0, pages past the table's
// width and page numbers outside the cache are skipped: nothing is written for them.
//
// Two kinds of cache:
//   * the inputs' type: rotate, round once, store; a warp per (token, heads), HBM-bound;
//   * e4m3 with a scale per (page, head) (e4m3.cuh). The scale needs the page's maximum before its first
//     code, so the unit of work is a request's page, some heads of k or v. A page whose first row is among the
//     new ones gets a fresh scale; another keeps its own unless the new rows need more, and then its
//     earlier rows move to the larger scale. Rows behind the last token are left alone.
//
// A page that receives tokens belongs to one request (shared prefix pages are full ones).
#include <algorithm>
#include <type_traits>

#include "e4m3.cuh"
#include "rope_common.cuh"

namespace msa {
namespace {

using namespace rope;

constexpr int kWarps = 8;
constexpr int kRowsPerLane = 4;
constexpr int kPageBlocks = 4;  // of the page kernel, to an SM (3: 67 us, 4: 62)
constexpr int kMaxDimFast = 256;

struct Half {  // k or v
  const void* x;
  void* cache;
  float* scale;
  int64_t x_ts, x_hs, c_ps, c_ts, c_hs;  // strides in elements
  int rotary;                            // 0 for v
};

struct Params {
  Half half[2];
  const float* table;
  const int32_t *cu, *block_table, *seq_lens;
  int64_t table_rows, tokens, num_pages;
  int batch, heads, dim, page_size, max_pages;
  FastDiv by_page, by_page_parts;  // page_size; items of a page
  uint32_t units, chunks, head_chunks;
  bool interleaved;
};

// Request of token t: the last b with cu[b] <= t; -1 before the first and behind the last.
__device__ __forceinline__ int request_of(const Params& p, int64_t t) {
  if (!p.cu) return (int)t;
  if (t < p.cu[0] || t >= p.cu[p.batch]) return -1;
  return find_sequence(p.cu, p.batch, t);
}

// Physical page of request b's logical page, or -1.
__device__ __forceinline__ int64_t physical_page(const Params& p, int b, int logical) {
  if (logical < 0 || logical >= p.max_pages) return -1;
  const int page = p.block_table[(int64_t)b * p.max_pages + logical];
  return page >= 0 && page < p.num_pages ? page : -1;
}

// New tokens of request b: rows [first, first + n), positions [pos, pos + n). Lengths and boundaries are 32-bit;
// what a broken cu_seqlens could overflow is 64.
struct Span {
  int64_t first;
  int pos, n;
};
__device__ __forceinline__ Span span_of(const Params& p, int b) {
  const int64_t begin = p.cu ? p.cu[b] : b, behind = p.cu ? p.cu[b + 1] : (int64_t)b + 1;
  int64_t first = begin, pos = (int64_t)p.seq_lens[b] - (behind - begin);
  if (pos < 0) first -= pos, pos = 0;  // tokens before position 0 are not stored
  if (first < 0) pos -= first, first = 0;
  const int64_t n = min(behind, p.tokens) - first;
  Span s;
  s.first = first;
  s.pos = (int)pos;
  s.n = n > 0 && pos + n <= 0x7fffffff ? (int)n : 0;
  return s;
}

// ------------------------------------------------------------------ caches in the inputs' type
template <typename T, int LPR, bool INTER>
__global__ void __launch_bounds__(kWarps * 32) append_kernel(const __grid_constant__ Params p) {
  constexpr int kSub = 32 / LPR;
  const uint32_t unit = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (unit >= p.units) return;
  const uint32_t t = unit / p.chunks;
  uint32_t chunk = unit - t * p.chunks;
  const bool is_v = chunk >= p.head_chunks;
  if (is_v) chunk -= p.head_chunks;
  const Half& s = p.half[is_v];
  const int lane = threadIdx.x & 31, l = lane % LPR;
  const LaneMap m = lane_map<INTER>(l, p.dim, s.rotary);
  const int h0 = chunk * (kSub * kRowsPerLane) + lane / LPR;
  const T* x = static_cast<const T*>(s.x) + (int64_t)t * s.x_ts;
  Raw<T> raw[kRowsPerLane][2];
#pragma unroll
  for (int i = 0; i < kRowsPerLane; ++i) {
    const int h = h0 + i * kSub;
    if (h < p.heads && m.active) {
      raw[i][0] = load_run(x + h * s.x_hs + m.a);
      raw[i][1] = load_run(x + h * s.x_hs + m.b);
    }
  }
  const int b = request_of(p, t);
  if (b < 0) return;
  const int64_t pos64 = (int64_t)p.seq_lens[b] - (p.cu ? (int64_t)p.cu[b + 1] - t : 1);
  if (pos64 < 0 || pos64 > 0x7fffffff) return;
  const int pos = (int)pos64, logical = p.by_page(pos);
  const int64_t page = physical_page(p, b, logical);
  if (page < 0) return;
  const bool rotated = m.rotated && s.rotary > 0, inside = s.rotary == 0 || pos < p.table_rows;
  float c[4], sn[4];
  if (inside && rotated) load_angles(p.table + (int64_t)pos * s.rotary, s.rotary, l, c, sn);
  T* out = static_cast<T*>(s.cache) + page * s.c_ps + (int64_t)(pos - logical * p.page_size) * s.c_ts;
#pragma unroll
  for (int i = 0; i < kRowsPerLane; ++i) {
    const int h = h0 + i * kSub;
    if (h >= p.heads || !m.active) continue;
    float v[8];
    unpack_lane<INTER>(raw[i], v);
    if (!inside) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = nan_f32();
    } else if (rotated) {
      rotate_lane(v, c, sn);
    }
    store_lane<INTER>(out + h * s.c_hs + m.a, out + h * s.c_hs + m.b, v);
  }
}

// ------------------------------------------------------------------ e4m3 caches
// The page task `task`: request, logical page and the new rows that fall into it. Request b's tasks
// start at cu[b] / S + 2 b: at least as many lie between two requests as the pages that n tokens can
// touch (n / S + 2), so a task finds its request by bisection without a scan over the requests.
struct Task {
  int64_t token;                     // row of k / v
  int b, logical, row_first, n, pos;  // request, logical page, first row in it, rows, position of the first
};
// False: nothing to do. The physical page is looked up apart (its loads would hold up the rows').
__device__ __forceinline__ bool find_task(const Params& p, int task, Task& r) {
  int b = task, index = 0;
  if (p.cu) {
    auto first_of = [&](int i) { return (int64_t)p.by_page(max(p.cu[i], 0)) + 2 * (int64_t)i; };
    int lo = 0, hi = p.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first_of(mid) <= task) lo = mid; else hi = mid - 1;
    }
    b = lo;
    const int64_t i = task - first_of(b);
    if (i < 0 || i >= p.max_pages) return false;
    index = (int)i;
  }
  const Span s = span_of(p, b);
  if (s.n <= 0) return false;
  const int logical = p.by_page(s.pos) + index;
  const int64_t page_begin = (int64_t)logical * p.page_size;
  const int64_t lo = max((int64_t)s.pos, page_begin), hi = min((int64_t)s.pos + s.n, page_begin + p.page_size);
  if (lo >= hi) return false;
  r.b = b;
  r.logical = logical;
  r.row_first = (int)(lo - page_begin);
  r.n = (int)(hi - lo);
  r.pos = (int)lo;
  r.token = s.first + (lo - s.pos);
  return true;
}

// Earlier rows of the page to the new scale, 16 codes a thread and step.
__device__ __forceinline__ void move_rows(uint8_t* page, int64_t row_stride, int rows, int dim, float ratio, int tid,
                                          int threads) {
  const int per = dim / 16;
#pragma unroll 8
  for (int i = tid; i < rows * per; i += threads) {
    uint4* at = reinterpret_cast<uint4*>(page + (int64_t)(i / per) * row_stride + (i % per) * 16);
    uint4 w = *at;
    w.x = e4m3::rescale4(w.x, ratio), w.y = e4m3::rescale4(w.y, ratio);
    w.z = e4m3::rescale4(w.z, ratio), w.w = e4m3::rescale4(w.w, ratio);
    *at = w;
  }
}

// New scale of the page, given its new rows' maximum.
__device__ __forceinline__ float grown_scale(float amax, int row_first, float old) {
  const float need = e4m3::scale_for(amax);
  return row_first == 0 ? need : fmaxf(old, need);
}

template <bool INTER>
__device__ __forceinline__ void store_codes(uint8_t* row, const LaneMap& m, const float (&v)[8], float inv) {
  uint32_t a, b;
  if (INTER) {
    a = e4m3::encode4(v[0], v[4], v[1], v[5], inv);
    b = e4m3::encode4(v[2], v[6], v[3], v[7], inv);
  } else {
    a = e4m3::encode4(v[0], v[1], v[2], v[3], inv);
    b = e4m3::encode4(v[4], v[5], v[6], v[7], inv);
  }
  *reinterpret_cast<uint32_t*>(row + m.a) = a;
  *reinterpret_cast<uint32_t*>(row + m.b) = b;
}

__device__ __forceinline__ float amax8(const float (&v)[8], float acc) {
#pragma unroll
  for (int i = 0; i < 8; ++i) acc = fmaxf(acc, e4m3::finite(v[i]) ? fabsf(v[i]) : 0.f);
  return acc;
}

// One row's eight values of a lane, rotated.
template <typename T, bool INTER>
__device__ __forceinline__ void rotated_row(const Params& p, const Half& s, const LaneMap& m, int l,
                                            const Raw<T> (&raw)[2], int64_t pos, float (&v)[8]) {
  unpack_lane<INTER>(raw, v);
  if (s.rotary == 0) return;
  if (pos >= p.table_rows) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = nan_f32();
  } else if (m.rotated) {
    float c[4], sn[4];
    load_angles(p.table + (int64_t)pos * s.rotary, s.rotary, l, c, sn);
    rotate_lane(v, c, sn);
  }
}

// One token per request: a warp per (request, head) of k or v.
template <typename T, int LPR, bool INTER>
__global__ void __launch_bounds__(kWarps * 32) append8_token_kernel(const __grid_constant__ Params p) {
  const uint32_t unit = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (unit >= p.units) return;
  const uint32_t rest = unit / p.heads;
  const int h = unit - rest * p.heads, b = rest / p.chunks;  // chunks: 2, or 1 without v
  const Half& s = p.half[rest - b * p.chunks];
  const int lane = threadIdx.x & 31, l = lane % LPR;
  const LaneMap m = lane_map<INTER>(l, p.dim, s.rotary);
  const bool mine = m.active && lane < LPR;
  const T* x = static_cast<const T*>(s.x) + (int64_t)b * s.x_ts + h * s.x_hs;
  Raw<T> raw[2] = {};
  if (mine) raw[0] = load_run(x + m.a), raw[1] = load_run(x + m.b);
  Task t;
  if (!find_task(p, (int)b, t)) return;
  const int64_t at = physical_page(p, t.b, t.logical);
  if (at < 0) return;
  float* scale = s.scale + at * p.heads + h;
  const float old = *scale;
  float v[8], amax = 0.f;
  rotated_row<T, INTER>(p, s, m, l, raw, t.pos, v);
  if (mine) amax = amax8(v, 0.f);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const float now = grown_scale(amax, t.row_first, old);
  uint8_t* page = static_cast<uint8_t*>(s.cache) + at * s.c_ps + h * s.c_hs;
  if (mine) store_codes<INTER>(page + t.row_first * s.c_ts, m, v, 1.f / now);
  if (t.row_first > 0 && now > old) move_rows(page, s.c_ts, (int)t.row_first, p.dim, old / now, lane, 32);
  if (lane == 0 && now != old) *scale = now;
}

__device__ __forceinline__ float block_amax(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) v = fmaxf(v, red[w]);
  return v;
}

// Chunks: a block takes HC heads (4, or 1 of a tensor with fewer) of a (request, page), of k or v. It reads the rows
// twice, once for the heads' maxima and once for the codes. That keeps whole kilobytes of a token's heads together and
// one set of angles for them, and holds nothing on the way. The second time the rows come from L2 as long as those of
// the blocks that run together fit it: four blocks an SM of 128 rows of 4 heads of 128 16-bit elements, 78 of its
// 126 MB. The maximum takes whatever is there: NaN drops out of fmaxf by itself, and only a page that holds an
// infinity is looked through again for its finite values.
// Measured: 32768 tokens, 8 heads of 128 (bf16), pages of 128: 60 us, 3.5 TB/s of the 210 MB that must move, 54% of
// the copy rate; DRAM reads are 1.1 times the input, so the second pass does hit L2. Issue slots are 66% busy:
// what is left is instructions (138 a lane for the two passes over a 16-byte piece). Where the blocks' rows outgrow L2,
// DRAM is read twice: float32 inputs (155 MB) 1.6 times the input, 90 us of a floor of 53; pages of 512 (264
// blocks, 138 MB) 1.8 times, 86 us of 32; both 2.0 times, 107 us of 53. A head at a time to a
// block, its rows held in registers or copied ahead into shared memory, took 75-93 us (256-byte pieces two
// kilobytes apart); eight heads 87 us (too few blocks).
template <typename T, int LPR, bool INTER, int HC>
__global__ void __launch_bounds__(kWarps * 32, kPageBlocks) append8_page_kernel(const __grid_constant__ Params p) {
  constexpr int kRows = kWarps * 32 / LPR;  // tokens of a step
  __shared__ float red[kWarps][HC], inverse[HC], ratio[HC];
  __shared__ bool infinite[HC];
  const int task = p.by_page_parts((int)blockIdx.x), part = (int)blockIdx.x - task * (int)(p.chunks * p.head_chunks);
  Task t;
  if (!find_task(p, task, t)) return;  // the same for the whole block
  const int64_t at = physical_page(p, t.b, t.logical);
  if (at < 0) return;
  const bool is_v = part >= (int)p.head_chunks;
  const Half& s = p.half[is_v];
  const int h0 = (part - is_v * (int)p.head_chunks) * HC, heads = min(HC, p.heads - h0);
  const int tid = threadIdx.x, l = tid % LPR, r0 = tid / LPR;
  const LaneMap m = lane_map<INTER>(l, p.dim, s.rotary);
  const bool turned = m.rotated && s.rotary > 0;
  // rows from here on have no angle
  const int inside = s.rotary > 0 ? (int)min(max(p.table_rows - t.pos, (int64_t)0), (int64_t)t.n) : t.n;
  float old = 0.f;
  if (tid < heads) old = s.scale[at * p.heads + h0 + tid];

  // Calls f(head, values, code row) for the lane's rotated values of every row.
  uint8_t* const page = static_cast<uint8_t*>(s.cache) + at * s.c_ps + h0 * s.c_hs;
  auto visit = [&](auto again, auto f) {
    const T* x = static_cast<const T*>(s.x) + (t.token + r0) * s.x_ts + h0 * s.x_hs + m.a;
    const int64_t to_b = m.b - m.a, step = kRows * s.x_ts, out_step = kRows * s.c_ts;
    const float* angle = turned ? p.table + (int64_t)(t.pos + r0) * s.rotary + kE * l : nullptr;
    uint8_t* out = page + (int64_t)(t.row_first + r0) * s.c_ts;
    for (int r = r0; r < t.n; r += kRows) {
      Raw<T> raw[HC][2];
      const T* row = x;
#pragma unroll
      for (int i = 0; i < HC; ++i) {
        raw[i][0].u = raw[i][1].u = {};
        if (i < heads && m.active) {
          raw[i][0] = again ? load_run_again(row) : load_run(row);
          raw[i][1] = again ? load_run_again(row + to_b) : load_run(row + to_b);
        }
        row += s.x_hs;
      }
      Angle2 angles;
      if (turned && r < inside) angles.load(angle, angle + s.rotary / 2);
      uint8_t* to = out;
#pragma unroll
      for (int i = 0; i < HC; ++i) {
        float v[2 * kE];
        unpack_lane<INTER>(raw[i], v);
        Lane y = lane_of(v);
        if (r >= inside) {
#pragma unroll
          for (int e = 0; e < kE; ++e) y.v[e] = twice(nan_f32());
        } else if (turned) {
          rotate_exact(y, angles);
        }
        if (i < heads && m.active) f(i, y, to);
        to += s.c_hs;
      }
      x += step;
      out += out_step;
      angle += kRows * s.rotary;
    }
  };
  // The heads' maxima, with or without infinite values, in red[0].
  auto maxima = [&](auto finite) {
    float amax[HC];
#pragma unroll
    for (int i = 0; i < HC; ++i) amax[i] = 0.f;
    visit(std::true_type(), [&](int i, const Lane& y, uint8_t*) {
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const float2 f = unpack2(y.v[e]);
        amax[i] = fmaxf(amax[i], finite && !e4m3::finite(f.x) ? 0.f : fabsf(f.x));
        amax[i] = fmaxf(amax[i], finite && !e4m3::finite(f.y) ? 0.f : fabsf(f.y));
      }
    });
#pragma unroll
    for (int i = 0; i < HC; ++i) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax[i] = fmaxf(amax[i], __shfl_xor_sync(0xffffffffu, amax[i], o));
      if ((tid & 31) == 0) red[tid >> 5][i] = amax[i];
    }
    __syncthreads();
    if (tid < HC) {
      float top = red[0][tid];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, red[w][tid]);
      red[0][tid] = top;
    }
    __syncthreads();
  };
  maxima(std::false_type());
  if (tid < HC) infinite[tid] = red[0][tid] == INFINITY;
  __syncthreads();
  bool any = false;
#pragma unroll
  for (int i = 0; i < HC; ++i) any = any || infinite[i];
  if (any) maxima(std::true_type());
  if (tid < heads) {
    const float now = grown_scale(red[0][tid], t.row_first, old);
    inverse[tid] = 1.f / now;
    ratio[tid] = t.row_first > 0 && now > old ? old / now : 1.f;
    if (now != old) s.scale[at * p.heads + h0 + tid] = now;
  }
  __syncthreads();
  float inv[HC];
#pragma unroll
  for (int i = 0; i < HC; ++i) inv[i] = i < heads ? inverse[i] : 0.f;
  visit(std::false_type(), [&](int i, const Lane& y, uint8_t* to) {
    float f[2 * kE], a[kE], b[kE];
    if (any) {
      floats_of(y, f);
      store_codes<INTER>(to, m, f, inv[i]);
      return;
    }
    Lane z;
#pragma unroll
    for (int e = 0; e < kE; ++e) z.v[e] = mul2(y.v[e], twice(inv[i]));
    floats_of(z, f);
    from_pairs<INTER>(f, a, b);
    *reinterpret_cast<uint32_t*>(to + m.a) = e4m3::encode2(a[0], a[1]) | e4m3::encode2(a[2], a[3]) << 16;
    *reinterpret_cast<uint32_t*>(to + m.b) = e4m3::encode2(b[0], b[1]) | e4m3::encode2(b[2], b[3]) << 16;
  });
  for (int i = 0; i < heads; ++i)
    if (ratio[i] != 1.f)
      move_rows(page + i * s.c_hs, s.c_ts, t.row_first, p.dim, ratio[i], tid, kWarps * 32);
}

// ------------------------------------------------------------------ any shape
// Unit by unit (pair or single element): head dims and rows off the vector layout, both kinds of cache.
// A block per (page task, head) of k or v.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) append_any_kernel(const __grid_constant__ Params p) {
  __shared__ float red[kWarps];
  Task t;
  if (!find_task(p, (int)blockIdx.x, t)) return;
  const int64_t at = physical_page(p, t.b, t.logical);
  if (at < 0) return;
  const int h = blockIdx.y;
  const Half& s = p.half[blockIdx.z];
  const int n_units = p.dim - s.rotary / 2;
  const int64_t n = t.n * n_units;
  const T* x = static_cast<const T*>(s.x) + t.token * s.x_ts + h * s.x_hs;
  auto value = [&](int64_t i, int64_t& row, Unit& e, float& a, float& b) {
    row = i / n_units;
    const int u = (int)(i - row * n_units);
    e = unit_of(u, s.rotary, p.interleaved);
    a = to_float(x[row * s.x_ts + e.a]);
    b = e.b >= 0 ? to_float(x[row * s.x_ts + e.b]) : 0.f;
    const int64_t pos = t.pos + row;
    if (s.rotary && pos >= p.table_rows) {
      a = b = nan_f32();
    } else if (e.b >= 0) {
      const float* angles = p.table + pos * s.rotary;
      rotate_pair(a, b, angles[u], angles[s.rotary / 2 + u]);
    }
  };
  int64_t row;
  Unit e;
  float a, b;
  if (!s.scale) {
    T* page = static_cast<T*>(s.cache) + at * s.c_ps + h * s.c_hs;
    for (int64_t i = threadIdx.x; i < n; i += kWarps * 32) {
      value(i, row, e, a, b);
      T* out = page + (t.row_first + row) * s.c_ts;
      out[e.a] = from_float<T>(a);
      if (e.b >= 0) out[e.b] = from_float<T>(b);
    }
    return;
  }
  float* scale = s.scale + at * p.heads + h;
  const float old = *scale;
  float amax = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += kWarps * 32) {
    value(i, row, e, a, b);
    amax = fmaxf(amax, fmaxf(e4m3::finite(a) ? fabsf(a) : 0.f, e4m3::finite(b) ? fabsf(b) : 0.f));
  }
  const float now = grown_scale(block_amax(amax, red), t.row_first, old), inv = 1.f / now;
  uint8_t* page = static_cast<uint8_t*>(s.cache) + at * s.c_ps + h * s.c_hs;
  for (int64_t i = threadIdx.x; i < n; i += kWarps * 32) {
    value(i, row, e, a, b);
    uint8_t* out = page + (t.row_first + row) * s.c_ts;
    out[e.a] = e4m3::encode1(a, inv);
    if (e.b >= 0) out[e.b] = e4m3::encode1(b, inv);
  }
  if (t.row_first > 0 && now > old)
    for (int64_t i = threadIdx.x; i < t.row_first * p.dim; i += kWarps * 32) {
      uint8_t* code = page + (i / p.dim) * s.c_ts + i % p.dim;
      *code = e4m3::encode1(e4m3::decode1(*code), old / now);
    }
  if (threadIdx.x == 0 && now != old) *scale = now;
}

// ------------------------------------------------------------------ host
bool fast_shape(const Params& p, int halves, int dtype, bool quantised) {
  if (p.dim % 8 || p.dim > kMaxDimFast || (quantised && p.dim % 16)) return false;
  if (reinterpret_cast<uintptr_t>(p.table) % 16) return false;
  const int es = elem_size(dtype);
  for (int i = 0; i < halves; ++i) {
    const Half& s = p.half[i];
    if (s.rotary % 8 || !rows_aligned(s.x, s.x_ts, s.x_hs, es, kE * es)) return false;
    if (quantised) {
      if (reinterpret_cast<uintptr_t>(s.cache) % 16 || s.c_ps % 16 || s.c_ts % 16 || s.c_hs % 16) return false;
    } else if (!rows_aligned(s.cache, s.c_ps, s.c_ts, es, kE * es) || s.c_hs % kE) {
      return false;
    }
  }
  return true;
}

template <typename T, int LPR, bool INTER>
void launch_fast(Params p, int halves, bool quantised, int64_t tasks, cudaStream_t st) {
  if (!quantised) {
    append_kernel<T, LPR, INTER><<<ceil_div(p.units, kWarps), kWarps * 32, 0, st>>>(p);
  } else if (!p.cu) {
    append8_token_kernel<T, LPR, INTER><<<ceil_div(p.units, kWarps), kWarps * 32, 0, st>>>(p);
  } else {
    const int together = p.heads >= 4 ? 4 : 1;
    p.chunks = halves;
    p.head_chunks = ceil_div(p.heads, together);
    const uint32_t parts = p.chunks * p.head_chunks;
    p.by_page_parts = FastDiv(parts);
    const unsigned blocks = (unsigned)(tasks * parts);
    if (together == 4) append8_page_kernel<T, LPR, INTER, 4><<<blocks, kWarps * 32, 0, st>>>(p);
    else append8_page_kernel<T, LPR, INTER, 1><<<blocks, kWarps * 32, 0, st>>>(p);
  }
}

template <typename T>
int launch(Params p, int halves, int dtype, bool quantised, cudaStream_t st) {
  // pages that the new tokens can touch, see find_task
  const int64_t tasks = p.cu ? p.tokens / p.page_size + 2 * (int64_t)p.batch : p.batch;
  MSA_CHECK_ARG(tasks * p.heads * halves < (int64_t)1 << 31 && p.heads <= 65535,
                "msa_cache_append: too many pages or heads");
  const bool fast = fast_shape(p, halves, dtype, quantised);
  // move_rows counts 16-byte units, append_any_kernel elements, of a head's page in 32 bits
  const int64_t page_elements = (int64_t)p.page_size * p.dim;
  MSA_CHECK_ARG(page_elements < (int64_t)1 << (!fast ? 31 : quantised ? 34 : 62),
                "msa_cache_append: page_size * head_dim is too large for this layout");
  if (fast) {
    const int lpr = p.dim <= 32 ? 4 : p.dim <= 64 ? 8 : p.dim <= 128 ? 16 : 32;
    p.head_chunks = ceil_div(p.heads, 32 / lpr * kRowsPerLane);
    p.chunks = quantised ? halves : p.head_chunks * halves;
    const int64_t units = quantised ? (int64_t)p.batch * p.heads * halves : p.tokens * p.chunks;
    MSA_CHECK_ARG(units < (int64_t)1 << 31, "msa_cache_append: too many tokens * heads");
    p.units = (uint32_t)units;
#define MSA_LAUNCH(LPR)                                                                   \
  if (p.interleaved) launch_fast<T, LPR, true>(p, halves, quantised, tasks, st);          \
  else launch_fast<T, LPR, false>(p, halves, quantised, tasks, st)
    switch (lpr) {
      case 4: MSA_LAUNCH(4); break;
      case 8: MSA_LAUNCH(8); break;
      case 16: MSA_LAUNCH(16); break;
      default: MSA_LAUNCH(32); break;
    }
#undef MSA_LAUNCH
  } else {
    append_any_kernel<T><<<dim3((unsigned)tasks, p.heads, halves), kWarps * 32, 0, st>>>(p);
  }
  count_launches(1);
  return launch_status("cache_append");
}

}  // namespace
}  // namespace msa

using namespace msa;

extern "C" int msa_cache_append(const void* k, const void* v, int dtype, int64_t k_token_stride,
                                int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                                const float* rope_table, int64_t table_rows, int32_t rotary_dim, int interleaved,
                                const int32_t* cu_seqlens, const int32_t* block_table, const int32_t* seq_lens,
                                int32_t batch, int64_t total_tokens, int32_t heads, int32_t head_dim,
                                int32_t page_size, int32_t max_pages, int64_t num_pages, void* k_cache, void* v_cache,
                                int cache_dtype, int64_t k_page_stride, int64_t k_slot_stride,
                                int64_t k_cache_head_stride, int64_t v_page_stride, int64_t v_slot_stride,
                                int64_t v_cache_head_stride, float* k_scale, float* v_scale, void* stream) {
  const bool quantised = cache_dtype == MSA_E4M3;
  MSA_CHECK_ARG(valid_dtype(dtype) && (quantised || cache_dtype == dtype), "msa_cache_append: bad dtype");
  MSA_CHECK_ARG(batch >= 0 && total_tokens >= 0 && heads >= 1 && head_dim >= 1 && page_size >= 1 && max_pages >= 0 &&
                    num_pages >= 0,
                "msa_cache_append: bad sizes");
  MSA_CHECK_ARG(cu_seqlens || total_tokens == batch, "msa_cache_append: without cu_seqlens one token per request");
  MSA_CHECK_ARG(rotary_dim >= 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim && table_rows >= 0 &&
                    (rotary_dim == 0 || table_rows == 0 || rope_table),  // an empty table has no address
                "msa_cache_append: rotary_dim must be even and at most head_dim, and needs a table");
  // nothing to store; empty tensors have no address
  if (batch == 0 || total_tokens == 0 || max_pages == 0 || num_pages == 0) return MSA_OK;
  MSA_CHECK_ARG(k && k_cache && block_table && seq_lens && !v == !v_cache,
                "msa_cache_append: missing pointers, or v without v_cache");
  MSA_CHECK_ARG(!quantised || (k_scale && (!v || v_scale)), "msa_cache_append: an e4m3 cache needs its scales");
  Params p{};
  p.half[0] = Half{k, k_cache, quantised ? k_scale : nullptr, k_token_stride, k_head_stride,
                   k_page_stride, k_slot_stride, k_cache_head_stride, rotary_dim};
  p.half[1] = Half{v, v_cache, quantised ? v_scale : nullptr, v_token_stride, v_head_stride,
                   v_page_stride, v_slot_stride, v_cache_head_stride, 0};
  p.table = rope_table, p.cu = cu_seqlens, p.block_table = block_table, p.seq_lens = seq_lens;
  p.table_rows = table_rows, p.tokens = total_tokens, p.num_pages = num_pages;
  p.batch = batch, p.heads = heads, p.dim = head_dim, p.page_size = page_size, p.max_pages = max_pages;
  p.by_page = FastDiv((uint32_t)page_size);
  p.interleaved = interleaved != 0;
  const int halves = v ? 2 : 1;
  cudaStream_t st = as_stream(stream);
  if (dtype == MSA_BF16) return launch<__nv_bfloat16>(p, halves, dtype, quantised, st);
  if (dtype == MSA_F16) return launch<__half>(p, halves, dtype, quantised, st);
  return launch<float>(p, halves, dtype, quantised, st);
}
