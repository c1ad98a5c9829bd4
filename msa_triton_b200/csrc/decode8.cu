// Decode attention over an 8-bit paged cache: decode.cu's semantics (one new token per request, its
// selected blocks of keys, a repeated block counts once, -1 pads) with e4m3 keys and values and one
// float32 scale per (page, head) for each (e4m3.cuh).
//
//   x_j = scale * log2(e) * ks[page(j)] * (q . kc_j)     out = sum_j 2^(x_j - M) vs[page(j)] vc_j / l
//   l = sum_j 2^(x_j - M)                                lse = (M + log2 l) ln 2
//
// HBM-bound: a key costs 2 D bytes and 4 h D flops for its group's h query heads. The work of a key is
// small but not free (each byte has to become a number), so both products run on mma.sync m16n8k16 (heads
// are the 16 rows; tcgen05's 128-row tiles would be 7/8 empty) and every byte is read from shared memory
// once, into the register that the instruction takes: no transposition.
//   * S = Q K^T: B's fragment wants pairs of neighbouring dims of one key; a lane (key n = lane / 4,
//     j = lane % 4) loads 16 bytes of its key's row, and the dims are renumbered so that its k index runs
//     over them (Q's fragment is renumbered the same way).
//   * O = P V: B's fragment wants pairs of neighbouring keys of one dim; a lane loads the same 16 dims of
//     the keys 2j, 2j + 1, 2j + 8, 2j + 9 and interleaves them two bytes at a time. The column of an
//     8-wide tile t is renumbered to dim 16 n + t.
// e4m3 fits fp16 exactly, so the operands are fp16: K and V exact; q divided by a power of two per head
// (exact but for elements 2^-14 below the head's largest, which keep 2^-25 of it); the weights rounded to
// 11 bits, which adds to a bf16 output less than its own rounding. float32 inputs take both q and the
// weights as a sum of two fp16 numbers. Accumulators, maxima and sums are float32.
//
// The values' scales vary by page, so the weights 2^(x_j) vs_j have a running maximum of their own (M' over
// x_j + log2 vs_j) beside the softmax's M: both stay in fp16's range whatever the scales are.
//
// A warp works on its own, 32 keys at a time, through a ring of kStages tiles in shared memory that
// cp.async fills (16 bytes a lane; the 16-byte units of a line are permuted so that neither product's
// reads meet a bank twice). Loads in flight cost no registers that way, and one address per key covers
// every page size and layout. The tiles of a (request, group) are dealt to the warps of a cluster of 1 to 8
// blocks, whose partial results are merged over distributed shared memory: one launch, no workspace.
#include <algorithm>

#include "e4m3.cuh"
#include "rope_common.cuh"

namespace msa {
namespace {

constexpr int kWarps = 4;
constexpr int kTile = 32;      // keys a warp takes at a time
constexpr int kStages = 2;
constexpr int kMaxSplits = 8;  // blocks of a cluster

struct Cache {
  const uint8_t* p;
  const float* scale;
  int64_t ps, ts, hs;  // page, token and head strides (bytes)
};

struct Params {
  const void* q;
  Cache k, v;
  const int32_t *block_table, *seq_lens, *ids;
  void* out;
  float* lse;
  int64_t num_pages;
  int q_heads, groups, dim, page_size, max_pages, topk, block, splits, dtype;
  float scale_log2;
};

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// With at most 8 heads the rows 8..15 are empty: their accumulators are never kept.
__device__ __forceinline__ void mma(float (&d)[2], uint32_t a0, uint32_t, uint32_t a2, uint32_t, uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "{\n\t.reg .f32 x, y;\n\t"
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, x, y}, {%2, %3, %4, %3}, {%5, %6}, "
      "{%0, %1, %7, %7};\n\t}"
      : "+f"(d[0]), "+f"(d[1])
      : "r"(a0), "r"(0), "r"(a2), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// What pack_half2 left over.
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t packed) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&packed));
  return pack_half2(a - f.x, b - f.y);
}

// Shared-memory offset of 16-byte unit `unit` of a tile's row. Keys are read four units of two
// neighbouring rows at a time, values one or two units of the rows 0, 2, 4, 6 (or 1, 3, 5, 7) apart.
template <int DP>
__device__ __forceinline__ uint32_t key_unit(int row, int unit) {
  const uint32_t at = row * DP + unit * 16;
  return DP == 64 ? at : at ^ ((row & 1) << 6);
}
template <int DP>
__device__ __forceinline__ uint32_t value_unit(int row, int unit) {
  return (row * DP + unit * 16) ^ (((row >> 1) & 3) << 5);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool wanted) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(wanted ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool wanted) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(wanted ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 u;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(at) : "memory");
  return u;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
  uint2 u;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(u.x), "=r"(u.y) : "r"(at) : "memory");
  return u;
}

// 16 bytes of a row from `d` on, one at a time, bytes past `dim` zero: rows off the 16-byte alignment.
__device__ __forceinline__ void copy_bytes(uint32_t dst, const uint8_t* row, int d, int dim, bool wanted) {
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    const uint32_t x = wanted && d + i < dim ? row[d + i] : 0;
    asm volatile("st.shared.u8 [%0], %1;" ::"r"(dst + i), "r"(x) : "memory");
  }
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
  if (dtype == MSA_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == MSA_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_any(void* p, int64_t i, int dtype, float x) {
  if (dtype == MSA_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else if (dtype == MSA_F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(x);
  else reinterpret_cast<float*>(p)[i] = x;
}

__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

__device__ __forceinline__ uint32_t cluster_address(uint32_t local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  return remote;
}
__device__ __forceinline__ float load_cluster(uint32_t at) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at));
  return x;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Bytes of a warp's shared memory: its ring (keys, values, their scales, the mask of each tile), its list
// of block ids; the partial result takes the same place at the end.
template <int DP, int HR>
struct Layout {
  static constexpr int kStage = 2 * kTile * DP + 2 * kTile * 4 + 16;
  static constexpr int kRing = kStages * kStage + 32 * 4;
  static constexpr int kRows = 8 * HR;
  static constexpr int kPart = (kRows * DP + 3 * kRows) * 4;
  static constexpr int kBytes = ((kRing > kPart ? kRing : kPart) + 127) / 128 * 128;
};

// DP: head dim rounded up to 64, 128 or 256. HR: head rows a lane holds (1: up to 8 heads, 2: up to 16).
// SPLIT: float32 inputs. VEC: rows are 16-byte aligned and dim is a multiple of 16 (other shapes all run the
// 16-row float32 form, which is right for every type and head count).
template <int DP, int HR, bool SPLIT, bool VEC>
__global__ void __launch_bounds__(kWarps * 32, DP == 128 && HR == 1 && !SPLIT ? 3 : 1)
decode8_kernel(const __grid_constant__ Params p) {
  using L = Layout<DP, HR>;
  constexpr int kSteps = DP / 16;   // k steps of S
  constexpr int kKC = DP / 64;      // 16-byte units of a key row per lane
  constexpr int kVB = DP / 8 < 16 ? DP / 8 : 16;  // bytes of a value row per lane and unit
  constexpr int kVC = DP / 8 / kVB;               // units
  constexpr int kTiles = DP / 8;                  // 8-wide output tiles
  constexpr int kKN = kTile / 8;                  // key groups of S
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, j = lane & 3;
  const int split = blockIdx.x % p.splits, bg = blockIdx.x / p.splits;
  const int b = bg / p.groups, g = bg - b * p.groups;
  const int h_all = p.q_heads / p.groups, h0 = blockIdx.y * 16, h = min(16, h_all - h0);
  const int pos = p.seq_lens[b] - 1;
  const int64_t q_row = (int64_t)b * p.q_heads + (int64_t)g * h_all + h0;
  // ---- queries: fragments of q / 2^e, and the factor 2^e * scale * log2(e) of each row
  uint32_t qa[HR][kSteps][2], qb[SPLIT ? HR : 1][SPLIT ? kSteps : 1][2];
  float qf[HR];
#pragma unroll
  for (int r = 0; r < HR; ++r) {
    const int head = n + 8 * r;
    float x[kKC][16], top = 0.f;
#pragma unroll
    for (int c = 0; c < kKC; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = 64 * c + 16 * j + i;
        x[c][i] = head < h && d < p.dim ? load_any(p.q, (q_row + head) * p.dim + d, p.dtype) : 0.f;
        top = fmaxf(top, fabsf(x[c][i]));
      }
    top = quad_max(top);
    // 2^e with top < 2^(e+1); nothing is scaled in an all-zero, subnormal or infinite row
    const uint32_t e = __float_as_uint(top) >> 23;
    const bool scaled = e >= 2 && e <= 252;
    const float inv = scaled ? __uint_as_float((254 - e) << 23) : 1.f;
    qf[r] = p.scale_log2 * (scaled ? __uint_as_float(e << 23) : 1.f);
#pragma unroll
    for (int c = 0; c < kKC; ++c)
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float a = x[c][4 * w + 2 * u] * inv, e2 = x[c][4 * w + 2 * u + 1] * inv;
          qa[r][4 * c + w][u] = pack_half2(a, e2);
          if (SPLIT) qb[r][4 * c + w][u] = pack_rest(a, e2, qa[r][4 * c + w][u]);
        }
  }
  // ---- running state
  float o[kTiles][2 * HR], m_soft[HR], m_val[HR], l[HR];
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int i = 0; i < 2 * HR; ++i) o[t][i] = 0.f;
#pragma unroll
  for (int r = 0; r < HR; ++r) m_soft[r] = m_val[r] = -INFINITY, l[r] = 0.f;

  uint8_t* mine = smem + warp * L::kBytes;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(mine);
  int32_t* slots = reinterpret_cast<int32_t*>(mine + kStages * L::kStage);  // this warp's compacted block ids
  const int per_block = (min(p.block, pos + 1) + kTile - 1) / kTile;
  const int warps = p.splits * kWarps;
  const int32_t* ids = p.ids + (int64_t)bg * p.topk;
  int before = 0;  // tiles of the earlier chunks of 32 ids
  for (int c0 = 0; c0 < p.topk && pos >= 0; c0 += 32) {
    const int id = c0 + lane < p.topk ? ids[c0 + lane] : -1;
    const uint32_t twins = __match_any_sync(0xffffffffu, id);
    bool valid = id >= 0 && id <= pos / p.block && (twins & ((1u << lane) - 1)) == 0;
    for (int i = 0; i < c0; ++i) valid = valid && ids[i] != id;
    const uint32_t chosen = __ballot_sync(0xffffffffu, valid);
    __syncwarp();
    if (valid) slots[__popc(chosen & ((1u << lane) - 1))] = id;
    __syncwarp();
    const int tiles = __popc(chosen) * per_block;
    const int first = (split * kWarps + warp + warps - before % warps) % warps;
    before += tiles;

    // Lane i looks up key i of a tile: its physical page (-1: no such key) and its row there.
    int page = -1, row_in_page = 0;
    auto look_up = [&](int tile) {
      page = -1;
      if (tile >= tiles) return;
      const int slot = tile / per_block, in_block = (tile - slot * per_block) * kTile + lane;
      const int64_t token = (int64_t)slots[slot] * p.block + in_block;
      if (in_block >= p.block || token > pos) return;
      const int logical = (int)token / p.page_size;  // token <= pos fits 32 bits
      row_in_page = (int)token - logical * p.page_size;
      if (logical < p.max_pages) page = p.block_table[(int64_t)b * p.max_pages + logical];
    };
    // Copies the tile that was looked up into a stage; always one group, empty behind the last tile.
    auto issue = [&](int stage) {
      const bool here = page >= 0 && page < p.num_pages;
      const uint32_t seen = __ballot_sync(0xffffffffu, here);
      const uint32_t base = ring + stage * L::kStage;
      if (seen) {
        const int64_t k_off = here ? page * p.k.ps + row_in_page * p.k.ts + g * p.k.hs : 0;
        const int64_t v_off = here ? page * p.v.ps + row_in_page * p.v.ts + g * p.v.hs : 0;
        constexpr int kUnits = DP / 16, kStep = 32 / kUnits;  // units of a row, rows of a step
        const int unit = lane % kUnits;
#pragma unroll(VEC ? kTile / kStep : 1)
        for (int i = 0; i < kTile / kStep; ++i) {
          const int row = i * kStep + lane / kUnits;
          const uint8_t* kr = p.k.p + __shfl_sync(0xffffffffu, k_off, row);
          const uint8_t* vr = p.v.p + __shfl_sync(0xffffffffu, v_off, row);
          const bool wanted = (seen >> row & 1) && unit * 16 < p.dim;
          const uint32_t kd = base + key_unit<DP>(row, unit), vd = base + kTile * DP + value_unit<DP>(row, unit);
          if (VEC) {
            cp_async16(kd, wanted ? kr + unit * 16 : p.k.p, wanted);
            cp_async16(vd, wanted ? vr + unit * 16 : p.v.p, wanted);
          } else {
            copy_bytes(kd, kr, unit * 16, p.dim, wanted);
            copy_bytes(vd, vr, unit * 16, p.dim, wanted);
          }
        }
        const int64_t at = here ? (int64_t)page * p.groups + g : 0;
        cp_async4(base + 2 * kTile * DP + 4 * lane, p.k.scale + at, here);
        cp_async4(base + 2 * kTile * DP + 4 * (kTile + lane), p.v.scale + at, here);
      }
      if (lane == 0) *reinterpret_cast<uint32_t*>(mine + stage * L::kStage + 2 * kTile * DP + 8 * kTile) = seen;
      cp_async_commit();
    };

    look_up(first);
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
      issue(s);
      look_up(first + (s + 1) * warps);
    }
    int stage = 0;
    for (int t = first; t < tiles; t += warps, stage = stage + 1 == kStages ? 0 : stage + 1) {
      issue(stage == 0 ? kStages - 1 : stage - 1);
      look_up(t + kStages * warps);
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const uint32_t base_k = ring + stage * L::kStage, base_v2 = base_k + kTile * DP;
      const float* scales = reinterpret_cast<const float*>(mine + stage * L::kStage + 2 * kTile * DP);
      const uint32_t now = *reinterpret_cast<const uint32_t*>(scales + 2 * kTile);
      if (now == 0) {  // no key of this tile is attended (behind the newest token)
        __syncwarp();
        continue;
      }
      // ---- S
      float x[kKN][2 * HR];
#pragma unroll
      for (int i = 0; i < kKN; ++i) {
#pragma unroll
        for (int e = 0; e < 2 * HR; ++e) x[i][e] = 0.f;
#pragma unroll
        for (int c = 0; c < kKC; ++c) {
          const uint4 unit = lds128(base_k + key_unit<DP>(8 * i + n, 4 * c + j));
          const uint32_t kw[4] = {unit.x, unit.y, unit.z, unit.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t b0 = e4m3::decode2((uint16_t)kw[w]), b1 = e4m3::decode2((uint16_t)(kw[w] >> 16));
            const int s = 4 * c + w;
            mma(x[i], qa[0][s][0], qa[HR - 1][s][0], qa[0][s][1], qa[HR - 1][s][1], b0, b1);
            if (SPLIT)
              mma(x[i], qb[0][SPLIT ? s : 0][0], qb[SPLIT ? HR - 1 : 0][SPLIT ? s : 0][0], qb[0][SPLIT ? s : 0][1],
                  qb[SPLIT ? HR - 1 : 0][SPLIT ? s : 0][1], b0, b1);
          }
        }
      }
      // ---- softmax weights
      float top[HR], top_v[HR];
#pragma unroll
      for (int r = 0; r < HR; ++r) top[r] = m_soft[r], top_v[r] = m_val[r];
      float shift[kKN][2];
#pragma unroll
      for (int i = 0; i < kKN; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = 8 * i + 2 * j + e;
          const float f = scales[key];
          shift[i][e] = log2f(scales[kTile + key]);
#pragma unroll
          for (int r = 0; r < HR; ++r) {
            float& y = x[i][2 * r + e];
            y = now >> key & 1 ? y * (qf[r] * f) : -INFINITY;
            top[r] = fmaxf(top[r], y);
            top_v[r] = fmaxf(top_v[r], y + shift[i][e]);
          }
        }
      float base[HR], base_v[HR], alpha_v[HR];
#pragma unroll
      for (int r = 0; r < HR; ++r) {
        top[r] = quad_max(top[r]);
        top_v[r] = quad_max(top_v[r]);
        base[r] = top[r] == -INFINITY ? 0.f : top[r];
        base_v[r] = top_v[r] == -INFINITY ? 0.f : top_v[r];
        l[r] *= exp2f(m_soft[r] - base[r]);
        alpha_v[r] = exp2f(m_val[r] - base_v[r]);
        m_soft[r] = top[r];
        m_val[r] = top_v[r];
      }
#pragma unroll
      for (int i = 0; i < kKN; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int r = 0; r < HR; ++r) {
            const float y = x[i][2 * r + e];
            l[r] += exp2f(y - base[r]);
            x[i][2 * r + e] = exp2f(y + shift[i][e] - base_v[r]);
          }
      bool rescale = false;
#pragma unroll
      for (int r = 0; r < HR; ++r) rescale = rescale || alpha_v[r] != 1.f;
      if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
        for (int d = 0; d < kTiles; ++d)
#pragma unroll
          for (int r = 0; r < HR; ++r) o[d][2 * r] *= alpha_v[r], o[d][2 * r + 1] *= alpha_v[r];
      }
      // ---- O += P V
#pragma unroll
      for (int s = 0; s < kTile / 16; ++s) {
        uint32_t a[4], rest[4] = {};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < HR; ++r) {
            const float y0 = x[2 * s + i][2 * r], y1 = x[2 * s + i][2 * r + 1];
            a[2 * i + r] = pack_half2(y0, y1);
            if (SPLIT) rest[2 * i + r] = pack_rest(y0, y1, a[2 * i + r]);
          }
        if (HR == 1) a[1] = a[3] = 0;
#pragma unroll
        for (int c = 0; c < kVC; ++c) {
          uint32_t vw[4][kVB / 4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = 16 * s + 2 * j + (i & 1) + 8 * (i >> 1);
            if constexpr (kVB == 16) {
              const uint4 u = lds128(base_v2 + value_unit<DP>(key, 8 * c + n));
              vw[i][0] = u.x, vw[i][1] = u.y, vw[i][2] = u.z, vw[i][3] = u.w;
            } else {
              const uint2 u = lds64(base_v2 + value_unit<DP>(key, n / 2) + (n & 1) * 8);
              vw[i][0] = u.x, vw[i][1] = u.y;
            }
          }
#pragma unroll
          for (int w = 0; w < kVB / 4; ++w) {
            // four dims of the keys (2j, 2j + 1) and (2j + 8, 2j + 9)
            const uint32_t lo0 = __byte_perm(vw[0][w], vw[1][w], 0x5140);
            const uint32_t lo1 = __byte_perm(vw[0][w], vw[1][w], 0x7362);
            const uint32_t hi0 = __byte_perm(vw[2][w], vw[3][w], 0x5140);
            const uint32_t hi1 = __byte_perm(vw[2][w], vw[3][w], 0x7362);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              const uint32_t lo = d < 2 ? lo0 : lo1, hi = d < 2 ? hi0 : hi1;
              const uint32_t b0 = e4m3::decode2((uint16_t)(d & 1 ? lo >> 16 : lo));
              const uint32_t b1 = e4m3::decode2((uint16_t)(d & 1 ? hi >> 16 : hi));
              const int tile = c * kVB + 4 * w + d;
              mma(o[tile], a[0], a[1], a[2], a[3], b0, b1);
              if (SPLIT) mma(o[tile], rest[0], rest[1], rest[2], rest[3], b0, b1);
            }
          }
        }
      }
      __syncwarp();  // the stage is free for the next copies
    }
    cp_async_wait<0>();
  }

  // ---- the warp's partial result to its shared memory: o[row][DP], then m_soft, m_val, l of its rows
  constexpr int kRows = L::kRows;
  __syncwarp();
  float* part = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int r = 0; r < HR; ++r) {
    const float sum = quad_sum(l[r]);
    const int row = n + 8 * r;
    if (j == 0) {
      part[kRows * DP + row] = m_soft[r];
      part[kRows * DP + kRows + row] = m_val[r];
      part[kRows * DP + 2 * kRows + row] = sum;
    }
    // column 2j + e of tile (c, t) is dim 128 c + kVB (2j + e) + t
#pragma unroll
    for (int c = 0; c < kVC; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < kVB; i += 4)
          *reinterpret_cast<float4*>(part + row * DP + 128 * c + kVB * (2 * j + e) + i) =
              make_float4(o[c * kVB + i][2 * r + e], o[c * kVB + i + 1][2 * r + e], o[c * kVB + i + 2][2 * r + e],
                          o[c * kVB + i + 3][2 * r + e]);
  }
  if (p.splits > 1) cluster_sync(); else __syncthreads();

  // ---- merge: the cluster's threads share the output elements
  const uint32_t here = (uint32_t)__cvta_generic_to_shared(smem);
  for (int i = split * kWarps * 32 + threadIdx.x; i < h * DP; i += p.splits * kWarps * 32) {
    const int row = i / DP, d = i - row * DP;
    float top = -INFINITY, top_v = -INFINITY, sum = 0.f, acc = 0.f;
    for (int s = 0; s < p.splits; ++s) {
      const uint32_t base = cluster_address(here, s);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const uint32_t at = base + w * L::kBytes + 4 * (kRows * DP + row);
        top = fmaxf(top, load_cluster(at));
        top_v = fmaxf(top_v, load_cluster(at + 4 * kRows));
      }
    }
    const float b0 = top == -INFINITY ? 0.f : top, bv = top_v == -INFINITY ? 0.f : top_v;
    for (int s = 0; s < p.splits; ++s) {
      const uint32_t base = cluster_address(here, s);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const uint32_t at = base + w * L::kBytes + 4 * (kRows * DP + row);
        sum += load_cluster(at + 8 * kRows) * exp2f(load_cluster(at) - b0);
        acc += load_cluster(base + w * L::kBytes + 4 * (row * DP + d)) * exp2f(load_cluster(at + 4 * kRows) - bv);
      }
    }
    // no key: zero and -inf; a NaN sum stays one
    const bool none = top == -INFINITY && sum == 0.f;
    if (d < p.dim)
      store_any(p.out, (q_row + row) * p.dim + d, p.dtype, none ? 0.f : acc * exp2f(bv - b0) / sum);
    if (d == 0) p.lse[q_row + row] = none ? -INFINITY : (b0 + log2f(sum)) * 0.6931471805599453f;
  }
  if (p.splits > 1) cluster_sync();  // the others may still read this block's memory
}

template <int DP, int HR, bool SPLIT, bool VEC>
int launch(const Params& p, int batch, cudaStream_t st) {
  const size_t smem = (size_t)kWarps * Layout<DP, HR>::kBytes;
  auto kernel = decode8_kernel<DP, HR, SPLIT, VEC>;
  if (smem > 48 * 1024)
    MSA_CUDA_RETURN(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(batch * p.groups * p.splits), (unsigned)ceil_div(p.q_heads / p.groups, 16));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {(unsigned)p.splits, 1, 1};
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  MSA_CUDA_RETURN(cudaLaunchKernelEx(&cfg, kernel, p));
  count_launches(1);
  return launch_status("decode_attn_e4m3");
}

template <int DP, int HR>
int launch_dim(const Params& p, int batch, bool vec, cudaStream_t st) {
  if (!vec) return launch<DP, 2, true, false>(p, batch, st);
  return p.dtype == MSA_F32 ? launch<DP, HR, true, true>(p, batch, st) : launch<DP, HR, false, true>(p, batch, st);
}

}  // namespace
}  // namespace msa

using namespace msa;

extern "C" int msa_decode_attn_e4m3(const void* q, int dtype, const void* k_cache, const void* v_cache,
                                    int64_t k_page_stride, int64_t k_slot_stride, int64_t k_head_stride,
                                    int64_t v_page_stride, int64_t v_slot_stride, int64_t v_head_stride,
                                    const float* k_scale, const float* v_scale, const int32_t* block_table,
                                    const int32_t* seq_lens, const int32_t* indices, int32_t batch, int32_t q_heads,
                                    int32_t groups, int32_t head_dim, int32_t page_size, int32_t max_pages,
                                    int64_t num_pages, int32_t topk_blocks, int32_t block_size, double scale,
                                    void* out, float* lse, void* stream) {
  MSA_CHECK_ARG(valid_dtype(dtype), "msa_decode_attn_e4m3: bad dtype");
  MSA_CHECK_ARG(groups >= 1 && q_heads >= 1 && q_heads % groups == 0,
                "msa_decode_attn_e4m3: q_heads must be a multiple of groups");
  MSA_CHECK_ARG(head_dim >= 1 && head_dim <= 256, "msa_decode_attn_e4m3: head_dim must be in [1, 256]");
  MSA_CHECK_ARG(page_size >= 1 && max_pages >= 0 && num_pages >= 0 && block_size >= 1 && topk_blocks >= 0 && batch >= 0,
                "msa_decode_attn_e4m3: bad sizes");
  MSA_CHECK_ARG((int64_t)batch * groups * kMaxSplits < (int64_t)1 << 31 && q_heads / groups <= 16 * 65535,
                "msa_decode_attn_e4m3: too many requests or heads");
  if (batch == 0) return MSA_OK;
  Params p{};
  p.q = q, p.dtype = dtype, p.out = out, p.lse = lse;
  p.k = Cache{static_cast<const uint8_t*>(k_cache), k_scale, k_page_stride, k_slot_stride, k_head_stride};
  p.v = Cache{static_cast<const uint8_t*>(v_cache), v_scale, v_page_stride, v_slot_stride, v_head_stride};
  p.block_table = block_table, p.seq_lens = seq_lens, p.ids = indices;
  p.num_pages = num_pages, p.q_heads = q_heads, p.groups = groups, p.dim = head_dim, p.page_size = page_size;
  p.max_pages = max_pages, p.topk = topk_blocks, p.block = block_size;
  p.scale_log2 = (float)(scale * 1.4426950408889634);
  // Blocks for a (request, group): until the chip is full, and no more warps than tiles.
  const int64_t tiles = (int64_t)topk_blocks * ((block_size + kTile - 1) / kTile);
  p.splits = 1;
  while (p.splits < kMaxSplits && (int64_t)batch * groups * p.splits < 148 * 6 && p.splits * kWarps < tiles) p.splits *= 2;
  const bool vec = head_dim % 16 == 0 && reinterpret_cast<uintptr_t>(k_cache) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(v_cache) % 16 == 0 &&
                   (k_page_stride | k_slot_stride | k_head_stride | v_page_stride | v_slot_stride | v_head_stride) % 16 == 0;
  cudaStream_t st = as_stream(stream);
  const bool few = q_heads / groups <= 8;
  if (head_dim <= 64) return few ? launch_dim<64, 1>(p, batch, vec, st) : launch_dim<64, 2>(p, batch, vec, st);
  if (head_dim <= 128) return few ? launch_dim<128, 1>(p, batch, vec, st) : launch_dim<128, 2>(p, batch, vec, st);
  return few ? launch_dim<256, 1>(p, batch, vec, st) : launch_dim<256, 2>(p, batch, vec, st);
}
