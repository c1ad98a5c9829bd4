// Decode attention over an 8-bit paged cache: decode.cu's semantics (one new token per request, its
// selected blocks of keys, a repeated block counts once, -1 pads) with e4m3 keys and values and one
// float32 scale per (page, head) for each (e4m3.cuh).
//
//   x_j = scale * log2(e) * ks[page(j)] * (q . kc_j)     out = sum_j 2^(x_j - M) vs[page(j)] vc_j / l
//   l = sum_j 2^(x_j - M)                                lse = (M + log2 l) ln 2
//
// HBM-bound: a key costs 2 D bytes and 4 h D flops for its group's h query heads. The work of a key is
// small but not free (each byte has to become a number), so both products run on mma.sync m16n8k16, keys
// or dims as the 16 rows and heads as the 8 columns (tcgen05's 128-row tiles would wait for 128 keys of one
// warp), and every byte is read from shared memory once, into the register that the instruction takes:
//   * S^T = K Q^T: A's fragment wants pairs of neighbouring dims of the keys n and n + 8; a lane (n = lane / 4,
//     j = lane % 4) reads 16 bytes of a key's row, and the dims are renumbered so that its k index runs
//     over them (Q's fragment is renumbered the same way).
//   * O^T = V^T P^T: A's fragment wants pairs of neighbouring keys of one dim; a lane reads the same 16 dims
//     of the keys 2j, 2j + 1, 2j + 8, 2j + 9 and interleaves them two bytes at a time. Rows n and n + 8 of
//     tile t are renumbered to the dims 16 n + 2 t and 16 n + 2 t + 1. P^T's fragment is S^T's after
//     movmatrix.
// e4m3 fits fp16 exactly, so the operands are fp16: K and V exact; q divided by a power of two per head
// (16-bit q exact but for elements 2^-14 below the head's largest, which keep 2^-25 of it; float32 q as a sum of two
// fp16 numbers); the weights as a sum of two fp16 numbers for every type, 2^-22 of a weight, so that an output's own
// rounding is the one that shows. (One fp16 number a weight: an fp16 output's error against float64 is 1.3 times
// that of float32 arithmetic, for 61.3 instead of 62.5 us at 64 requests, 393 instead of 401 us at 256 long ones.)
// Accumulators, maxima and sums are float32.
//
// The values' scales vary by page, so the weights 2^(x_j) vs_j have a reference of their own beside the softmax's M.
// With vs_j = 2^e_j m_j, 1 <= m_j < 2, they are 2^(x_j - M + e_j - M') m_j, M' an integer near the maximum of
// x_j - M + e_j: everything in the exponent but x_j - M is exact, however large the logits and far apart the scales (a
// logarithm of vs_j added to a logit of 1000 would keep 2^-15). Neither M nor M' has to be the maximum itself: they
// move, with the shuffles and the scaling that takes, only once a key lies more than kSlack above one of them.
// Weights enter the products 2^kLift higher (taken off the output again): below 2^(kLift + kSlack + 1) < 2^16 in
// fp16's range, so that what fp16 loses at its lower end, 2^-25, is 2^-38 of the row's largest weight times value scale.
// Weights up to 1 would lose 2^-25 of it, and the sum of many keys far below the largest with them.
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
constexpr int kStages = 2;     // tiles of a warp's ring
constexpr int kMaxSplits = 8;  // blocks of a cluster
constexpr int kLift = 13;      // see above; kLift + kSlack + 1 stays below 16
constexpr float kSlack = 1.9f;

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
  int q_heads, groups, dim, page_size, max_pages, topk, block, dtype;
  // Clusters of 2^split_shift blocks. The first `shared` items ((request, group) pairs) take a cluster each, those
  // after them a block each.
  int split_shift, shared;
  FastDiv by_page;
  float scale_log2;
  bool uniform;  // 16 keys in a row never leave a page
};

// (Neither this nor movmatrix is volatile: what they give depends on their operands alone, and in a fixed order
// they cost registers that spill: 63.5 instead of 61.3 us at 64 requests.)
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The transposed 8 x 8 matrix of 16-bit elements, row lane / 4, columns 2 (lane % 4) and the next.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
               : "r"(at)
               : "memory");
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

// 16 elements of a row from `d` on as floats, those past `dim` (or of an unwanted row) zero. VEC: 16-byte loads.
template <bool VEC>
__device__ __forceinline__ void load_q(float (&x)[16], const void* q, int64_t row, int d, int dim, int dtype,
                                       bool wanted) {
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.f;
  if (!wanted || d >= dim) return;
  if (!VEC) {
    for (int i = 0; i < 16 && d + i < dim; ++i) {
      const int64_t at = row * dim + d + i;
      x[i] = dtype == MSA_BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(q)[at])
             : dtype == MSA_F16 ? __half2float(reinterpret_cast<const __half*>(q)[at])
                                : reinterpret_cast<const float*>(q)[at];
    }
    return;
  }
  const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(q) +
                                                     (row * dim + d) * (dtype == MSA_F32 ? 4 : 2));
  uint4 u[4];
  u[0] = __ldg(from), u[1] = __ldg(from + 1);
  if (dtype == MSA_F32) {
    u[2] = __ldg(from + 2), u[3] = __ldg(from + 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[4 * i] = __uint_as_float(u[i].x), x[4 * i + 1] = __uint_as_float(u[i].y);
      x[4 * i + 2] = __uint_as_float(u[i].z), x[4 * i + 3] = __uint_as_float(u[i].w);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w = i & 3 ? (i & 3) == 1 ? u[i / 4].y : (i & 3) == 2 ? u[i / 4].z : u[i / 4].w : u[i / 4].x;
    const float2 f = dtype == MSA_BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w))
                                       : __half22float2(*reinterpret_cast<const __half2*>(&w));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}

// Four elements of the output from `d` on.
template <bool VEC>
__device__ __forceinline__ void store_out(void* out, int64_t row, int d, int dim, int dtype, float4 v) {
  if (d >= dim) return;
  const int64_t at = row * dim + d;
  const float f[4] = {v.x, v.y, v.z, v.w};
  if (VEC) {
    if (dtype == MSA_BF16) rope::store_run(reinterpret_cast<__nv_bfloat16*>(out) + at, f);
    else if (dtype == MSA_F16) rope::store_run(reinterpret_cast<__half*>(out) + at, f);
    else rope::store_run(reinterpret_cast<float*>(out) + at, f);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (d + e < dim) {
      if (dtype == MSA_BF16) reinterpret_cast<__nv_bfloat16*>(out)[at + e] = __float2bfloat16_rn(f[e]);
      else if (dtype == MSA_F16) reinterpret_cast<__half*>(out)[at + e] = __float2half_rn(f[e]);
      else reinterpret_cast<float*>(out)[at + e] = f[e];
    }
}

// 2^x by the special function unit (2 ulp; a subnormal result, a weight 2^-126 of the largest, is zero).
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Over the eight lanes that share lane % 4.
__device__ __forceinline__ float column_max(float x) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float column_sum(float x) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

__device__ __forceinline__ uint32_t cluster_address(uint32_t local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  return remote;
}
__device__ __forceinline__ void store_cluster4(uint32_t at, float4 x) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(x.x), "f"(x.y), "f"(x.z), "f"(x.w)
               : "memory");
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Bytes of a warp's shared memory: its ring (keys, values, four floats a key: its scale, the value's, and that one's
// exponent and mantissa once they are split; the mask of each tile), its list of block ids; the partial result takes
// the same place at the end.
template <int DP, int HR>
struct Layout {
  static constexpr int kStage = 2 * kTile * DP + kTile * 16 + 16;
  static constexpr int kRing = kStages * kStage + 32 * 4;
  static constexpr int kRows = 8 * HR;
  static constexpr int kPitch = DP + 4;  // floats; with part_at, no bank twice when a warp stores its rows
  static constexpr int kStats = kRows * kPitch;  // then m_soft, m_val, l of each row
  static constexpr int kPart = (kStats + 3 * kRows) * 4;
  static constexpr int kBytes = ((kRing > kPart ? kRing : kPart) + 127) / 128 * 128;
  // what the cluster's blocks send one another: their shares of o, then (m_soft, m_val, l, -) of each row
  static constexpr int kInbox = kRows * DP * 4 + kMaxSplits * kRows * 16;
};

// Float offset of the four dims 4 i .. 4 i + 3 of a row of the partial result.
template <int DP, int HR>
__device__ __forceinline__ int part_at(int row, int i) {
  return row * Layout<DP, HR>::kPitch + 4 * (i ^ ((i >> 2) & 1));
}

// DP: head dim rounded up to 64, 128 or 256. HR: tiles of 8 heads (1 or 2).
// SPLIT: float32 inputs (q in two terms). VEC: rows (q's and out's too) are 16-byte aligned and dim is a multiple of 16 (other
// shapes all run the 16-row float32 form, which is right for every type and head count).
template <int DP, int HR, bool SPLIT, bool VEC>
__global__ void __launch_bounds__(kWarps * 32, DP == 128 && HR == 1 && !SPLIT ? 3 : 1)
decode8_kernel(const __grid_constant__ Params p) {
  using L = Layout<DP, HR>;
  constexpr int kSteps = DP / 16;   // k steps of S
  constexpr int kKC = DP / 64;      // 16-byte units of a key row per lane
  constexpr int kVB = DP / 8 < 16 ? DP / 8 : 16;  // bytes of a value row per lane and unit
  constexpr int kVC = DP / 8 / kVB;               // units
  constexpr int kTiles = DP / 16;                 // 16-dim output tiles
  constexpr int kKT = kTile / 16;                 // 16-key tiles of S
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, j = lane & 3;
  const int shared_blocks = p.shared << p.split_shift, behind = (int)blockIdx.x - shared_blocks;
  const int split_shift = behind >= 0 ? 0 : p.split_shift, splits = 1 << split_shift;  // the same for a whole cluster
  const int split = behind >= 0 ? 0 : blockIdx.x & (splits - 1);
  const int bg = behind >= 0 ? p.shared + behind : blockIdx.x >> split_shift;
  const int b = bg / p.groups, g = bg - b * p.groups;
  const int h_all = p.q_heads / p.groups, h0 = blockIdx.y * 16, h = min(16, h_all - h0);
  if (splits > 1) cluster_arrive();  // waited for before the first store to another block
  const int32_t* ids = p.ids + (int64_t)bg * p.topk;
  int id = lane < p.topk ? ids[lane] : -1;
  const int pos = p.seq_lens[b] - 1;
  const int64_t q_row = (int64_t)b * p.q_heads + (int64_t)g * h_all + h0;
  // ---- queries: fragments of q / 2^e, and the factor 2^e of each row
  // (read after the first copies are on their way)
  uint32_t qa[HR][kSteps][2] = {}, qb[SPLIT ? HR : 1][SPLIT ? kSteps : 1][2] = {};
  float qf[HR][2] = {};  // of the heads 8 r + 2 j + e, the columns of this lane
  auto load_queries = [&]() {
#pragma unroll
    for (int r = 0; r < HR; ++r) {
      const int head = n + 8 * r;
      float x[kKC][16], top = 0.f;
#pragma unroll
      for (int c = 0; c < kKC; ++c) {
        load_q<VEC>(x[c], p.q, q_row + head, 64 * c + 16 * j, p.dim, p.dtype, head < h);
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[c][i]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e with top < 2^(e+1), or < 2^(e+2) at the range's upper end; subnormal rows come out below 1, with all the
      // bits that they have
      const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 253u);
      const float inv = __uint_as_float((254 - e) << 23), f = __uint_as_float(e << 23);
      qf[r][0] = __shfl_sync(0xffffffffu, f, 8 * j);
      qf[r][1] = __shfl_sync(0xffffffffu, f, 8 * j + 4);
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
  };
  // ---- running state
  float o[HR][kTiles][4], m_soft[HR][2], m_val[HR][2], l[HR][2];
#pragma unroll
  for (int r = 0; r < HR; ++r) {
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[r][t][i] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) m_soft[r][e] = m_val[r][e] = -INFINITY, l[r][e] = 0.f;
  }

  uint8_t* mine = smem + warp * L::kBytes;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(mine);
  int32_t* slots = reinterpret_cast<int32_t*>(mine + kStages * L::kStage);  // this warp's compacted block ids
  const int per_block = (min(p.block, pos + 1) + kTile - 1) / kTile;
  const int warps = splits * kWarps;
  int before = 0;  // tiles of the earlier chunks of 32 ids
  for (int c0 = 0; c0 < p.topk && pos >= 0; c0 += 32) {
    if (c0) id = c0 + lane < p.topk ? ids[c0 + lane] : -1;
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
    struct Row {
      int page, row;
    };
    auto look_up = [&](int tile) {
      Row r{-1, 0};
      if (tile >= tiles) return r;
      const int slot = tile / per_block, in_block = (tile - slot * per_block) * kTile + lane;
      const int64_t token = (int64_t)slots[slot] * p.block + in_block;
      if (in_block >= p.block || token > pos) return r;
      const int logical = p.by_page((int)token);  // token <= pos fits 32 bits
      r.row = (int)token - logical * p.page_size;
      if (logical < p.max_pages) r.page = p.block_table[(int64_t)b * p.max_pages + logical];
      return r;
    };
    // Copies a tile that was looked up into a stage; always one group, empty behind the last tile.
    auto issue = [&](int stage, const Row& r) {
      const int page = r.page, row_in_page = r.row;
      const bool here = page >= 0 && page < p.num_pages;
      const uint32_t seen = __ballot_sync(0xffffffffu, here);
      const uint32_t base = ring + stage * L::kStage;
      if (seen) {
        const int64_t k_off = here ? page * p.k.ps + row_in_page * p.k.ts + g * p.k.hs : 0;
        const int64_t v_off = here ? page * p.v.ps + row_in_page * p.v.ts + g * p.v.hs : 0;
        constexpr int kUnits = DP / 16, kStep = 32 / kUnits;  // units of a row, rows of a step
        const int unit = lane % kUnits, sub = lane / kUnits;
        if (VEC && p.uniform && seen == 0xffffffffu) {
          // two runs of 16 rows, each at a fixed stride
          const bool inside = unit * 16 < p.dim;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const uint8_t* kr = p.k.p + __shfl_sync(0xffffffffu, k_off, 16 * s) + sub * p.k.ts + unit * 16;
            const uint8_t* vr = p.v.p + __shfl_sync(0xffffffffu, v_off, 16 * s) + sub * p.v.ts + unit * 16;
#pragma unroll
            for (int i = 0; i < 16 / kStep; ++i) {
              const int row = 16 * s + i * kStep + sub;
              cp_async16(base + key_unit<DP>(row, unit), inside ? kr : p.k.p, inside);
              cp_async16(base + kTile * DP + value_unit<DP>(row, unit), inside ? vr : p.v.p, inside);
              kr += kStep * p.k.ts;
              vr += kStep * p.v.ts;
            }
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < kTile / kStep; ++i) {
            const int row = i * kStep + sub;
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
        }
        const int64_t at = here ? (int64_t)page * p.groups + g : 0;
        cp_async4(base + 2 * kTile * DP + 16 * lane, p.k.scale + at, here);
        cp_async4(base + 2 * kTile * DP + 16 * lane + 4, p.v.scale + at, here);
      }
      if (lane == 0) *reinterpret_cast<uint32_t*>(mine + stage * L::kStage + 2 * kTile * DP + 16 * kTile) = seen;
      cp_async_commit();
    };

    // the table is read a tile ahead of the copies, the copies a tile ahead of the products
    const Row now_row = look_up(first);
    Row next = look_up(first + warps);
    issue(0, now_row);
    if (c0 == 0) load_queries();
    int stage = 0;
    for (int t = first; t < tiles; t += warps, stage ^= 1) {
      issue(stage ^ 1, next);
      next = look_up(t + 2 * warps);
      cp_async_wait<1>();
      __syncwarp();
      const uint32_t base_k = ring + stage * L::kStage, base_v2 = base_k + kTile * DP;
      float* scales = reinterpret_cast<float*>(mine + stage * L::kStage + 2 * kTile * DP);
      const uint32_t now = *reinterpret_cast<const uint32_t*>(scales + 4 * kTile);
      if (now == 0) {  // no key of this tile is attended (behind the newest token)
        __syncwarp();
        continue;
      }
      {  // the key scale times scale * log2(e); the value scale as 2^e m, m times 2^kLift (zero and subnormal ones have
         // e = -126)
        const float s = scales[4 * lane + 1];
        const int e = min(max((int)(__float_as_uint(s) >> 23 & 255), 1), 254);
        *reinterpret_cast<float4*>(scales + 4 * lane) =
            make_float4(scales[4 * lane] * p.scale_log2, s, (float)(e - 127),
                        s * __uint_as_float(max((254u - e) << 23, 0x400000u)) * (1 << kLift));
      }
      __syncwarp();
      // ---- S^T: x[kt][r][2 a + e] is key 16 kt + n + 8 a, head 8 r + 2 j + e
      float x[kKT][HR][4];
#pragma unroll
      for (int kt = 0; kt < kKT; ++kt) {
#pragma unroll
        for (int r = 0; r < HR; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[kt][r][i] = 0.f;
#pragma unroll
        for (int c = 0; c < kKC; ++c) {
          const uint4 u0 = lds128(base_k + key_unit<DP>(16 * kt + n, 4 * c + j));
          const uint4 u1 = lds128(base_k + key_unit<DP>(16 * kt + n + 8, 4 * c + j));
          const uint32_t w0[4] = {u0.x, u0.y, u0.z, u0.w}, w1[4] = {u1.x, u1.y, u1.z, u1.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t a0, a1, a2, a3;
            e4m3::decode4(w0[w], a0, a2);
            e4m3::decode4(w1[w], a1, a3);
            const int s = 4 * c + w;
#pragma unroll
            for (int r = 0; r < HR; ++r) {
              mma(x[kt][r], a0, a1, a2, a3, qa[r][s][0], qa[r][s][1]);
              if (SPLIT) {
                const uint32_t(&rest)[2] = qb[SPLIT ? r : 0][SPLIT ? s : 0];
                mma(x[kt][r], a0, a1, a2, a3, rest[0], rest[1]);
              }
            }
          }
        }
      }
      // ---- softmax weights
      float top[HR][2], top_v[HR][2], base[HR][2], shift[kKT][2], mantissa[kKT][2];
#pragma unroll
      for (int r = 0; r < HR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[r][e] = top_v[r][e] = -INFINITY;
          base[r][e] = m_soft[r][e] == -INFINITY ? 0.f : m_soft[r][e];
        }
#pragma unroll
      for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const int key = 16 * kt + n + 8 * a;
          const float4 of = *reinterpret_cast<const float4*>(scales + 4 * key);
          const float f = of.x;
          shift[kt][a] = of.z;
          mantissa[kt][a] = of.w;
#pragma unroll
          for (int r = 0; r < HR; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) x[kt][r][2 * a + e] *= qf[r][e] * f;
        }
      if (now != 0xffffffffu) {
#pragma unroll
        for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
          for (int a = 0; a < 2; ++a)
            if (!(now >> (16 * kt + n + 8 * a) & 1)) {
#pragma unroll
              for (int r = 0; r < HR; ++r) x[kt][r][2 * a] = x[kt][r][2 * a + 1] = -INFINITY;
            }
      }
      bool grown = false;
#pragma unroll
      for (int r = 0; r < HR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
            for (int a = 0; a < 2; ++a) {
              const float y = x[kt][r][2 * a + e];
              top[r][e] = fmaxf(top[r][e], y);
              top_v[r][e] = fmaxf(top_v[r][e], y - base[r][e] + shift[kt][a]);
            }
          grown = grown || top[r][e] > m_soft[r][e] + kSlack || top_v[r][e] > m_val[r][e] + kSlack;
        }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int r = 0; r < HR; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float ms = fmaxf(m_soft[r][e], column_max(top[r][e]));
            base[r][e] = ms == -INFINITY ? 0.f : ms;
            const float delta = m_soft[r][e] - base[r][e];
            m_soft[r][e] = ms;
            l[r][e] *= fast_exp2(delta);
            float tv = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
              for (int a = 0; a < 2; ++a) tv = fmaxf(tv, x[kt][r][2 * a + e] - base[r][e] + shift[kt][a]);
            // m_val is relative to m_soft
            const float before = m_val[r][e] + delta, mv = floorf(fmaxf(before, column_max(tv)));
            const float alpha = fast_exp2(before - (mv == -INFINITY ? 0.f : mv));
            m_val[r][e] = mv;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) o[r][t][e] *= alpha, o[r][t][2 + e] *= alpha;
          }
      }
#pragma unroll
      for (int r = 0; r < HR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float base_v = m_val[r][e] == -INFINITY ? 0.f : m_val[r][e];
#pragma unroll
          for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
            for (int a = 0; a < 2; ++a) {
              const float y = x[kt][r][2 * a + e] - base[r][e];
              l[r][e] += fast_exp2(y);
              x[kt][r][2 * a + e] = fast_exp2(y + (shift[kt][a] - base_v)) * mantissa[kt][a];
            }
        }
      // ---- O^T += V^T P^T
#pragma unroll
      for (int s = 0; s < kKT; ++s) {
        uint32_t b[HR][2], rest[HR][2];
#pragma unroll
        for (int r = 0; r < HR; ++r)
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            const float y0 = x[s][r][2 * a], y1 = x[s][r][2 * a + 1];
            const uint32_t packed = pack_half2(y0, y1);
            b[r][a] = transpose8(packed);
            rest[r][a] = transpose8(pack_rest(y0, y1, packed));
          }
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
            // four dims of the keys (2j, 2j + 1) and (2j + 8, 2j + 9): two tiles
            uint32_t a[2][4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t pick = half ? 0x7362 : 0x5140;
              e4m3::decode4(__byte_perm(vw[0][w], vw[1][w], pick), a[half][0], a[half][1]);
              e4m3::decode4(__byte_perm(vw[2][w], vw[3][w], pick), a[half][2], a[half][3]);
            }
            // the tiles in turn: the second term of one would wait for its first
#pragma unroll
            for (int term = 0; term < 2; ++term)
#pragma unroll
              for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int r = 0; r < HR; ++r) {
                  const uint32_t(&weights)[2] = term ? rest[r] : b[r];
                  mma(o[r][c * (kVB / 2) + 2 * w + half], a[half][0], a[half][1], a[half][2], a[half][3], weights[0],
                      weights[1]);
                }
          }
        }
      }
      __syncwarp();  // the stage is free for the next copies
    }
    cp_async_wait<0>();
  }

  // ---- the warp's partial result to its shared memory
  constexpr int kRows = L::kRows;
  __syncwarp();
  float* part = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int r = 0; r < HR; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float sum = column_sum(l[r][e]);
      const int row = 8 * r + 2 * j + e;
      if (n == 0) {
        part[L::kStats + row] = m_soft[r][e];
        part[L::kStats + kRows + row] = m_val[r][e];
        part[L::kStats + 2 * kRows + row] = sum;
      }
      // rows n and n + 8 of tile (c, t) are the dims 128 c + kVB n + 2 t and the next
#pragma unroll
      for (int c = 0; c < kVC; ++c)
#pragma unroll
        for (int i = 0; i < kVB / 2; i += 2) {
          const int t = c * (kVB / 2) + i;
          *reinterpret_cast<float4*>(part + part_at<DP, HR>(row, (128 * c + kVB * n + 2 * i) / 4)) =
              make_float4(o[r][t][e], o[r][t][2 + e], o[r][t + 1][e], o[r][t + 1][2 + e]);
        }
    }
  __syncthreads();

  // m: the softmax's reference; mv: the values', relative to it
  auto finish = [&](int row, int i, float m, float mv, float sum, float4 acc) {
    // no key: zero and -inf; a NaN sum stays one
    const bool none = m == -INFINITY && sum == 0.f;
    // the sum and 2^kLift first: the product stays near the codes, whatever the scales are
    const float f = exp2f(mv), g = 1.f / (1 << kLift) / sum;
    store_out<VEC>(p.out, q_row + row, 4 * i, p.dim, p.dtype,
                   none ? make_float4(0.f, 0.f, 0.f, 0.f)
                        : make_float4(acc.x * g * f, acc.y * g * f, acc.z * g * f, acc.w * g * f));
    if (i == 0) p.lse[q_row + row] = none ? -INFINITY : ((m == -INFINITY ? 0.f : m) + log2f(sum)) * 0.6931471805599453f;
  };
  auto add = [](float4& acc, const float4& v, float f) {
    acc.x = fmaf(v.x, f, acc.x), acc.y = fmaf(v.y, f, acc.y), acc.z = fmaf(v.z, f, acc.z), acc.w = fmaf(v.w, f, acc.w);
  };

  // ---- join the block's warps, four output elements a thread; with more blocks, send them to the block
  // that finishes them (element at: block at % splits)
  const uint32_t inbox = (uint32_t)__cvta_generic_to_shared(smem) + kWarps * L::kBytes;
  const uint32_t inbox_stats = inbox + kRows * DP * 4;
  const int elements = h * (DP / 4), share = elements >> split_shift;  // DP / 4 is a multiple of kMaxSplits
  if (splits > 1) cluster_wait();  // every block of the cluster has started: its memory may be written
  for (int at = threadIdx.x; at < elements; at += kWarps * 32) {
    const int row = at / (DP / 4), i = at % (DP / 4);
    float m = -INFINITY, mv = -INFINITY, sum = 0.f, ms[kWarps], mvs[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float* stats = reinterpret_cast<const float*>(smem + w * L::kBytes) + L::kStats + row;
      ms[w] = stats[0], mvs[w] = stats[kRows];
      m = fmaxf(m, ms[w]);
    }
    const float m0 = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      mvs[w] += ms[w] - m0;  // relative to the common maximum
      mv = fmaxf(mv, mvs[w]);
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float* from = reinterpret_cast<const float*>(smem + w * L::kBytes);
      sum += from[L::kStats + 2 * kRows + row] * fast_exp2(ms[w] - m0);
      add(acc, *reinterpret_cast<const float4*>(from + part_at<DP, HR>(row, i)),
          fast_exp2(mvs[w] - (mv == -INFINITY ? 0.f : mv)));
    }
    if (splits == 1) {
      finish(row, i, m, mv, sum, acc);
    } else {
      store_cluster4(cluster_address(inbox, at & (splits - 1)) + 16 * (split * share + (at >> split_shift)), acc);
      if (i < splits)
        store_cluster4(cluster_address(inbox_stats, i) + 16 * (split * kRows + row), make_float4(m, mv, sum, 0.f));
    }
  }
  if (splits == 1) return;

  // ---- this block's elements, from its own memory: nobody reads it any more after this
  __syncwarp();  // the cluster barrier takes whole warps
  cluster_arrive();
  cluster_wait();
  const float4* shares = reinterpret_cast<const float4*>(smem + kWarps * L::kBytes);
  const float4* stats = shares + kRows * DP / 4;
  for (int k = threadIdx.x; k < share; k += kWarps * 32) {
    const int at = (k << split_shift) + split, row = at / (DP / 4), i = at % (DP / 4);
    float4 part[kMaxSplits], s[kMaxSplits];
    float m = -INFINITY, mv = -INFINITY, sum = 0.f;
#pragma unroll
    for (int r = 0; r < kMaxSplits; ++r) {
      const int from = min(r, splits - 1);
      s[r] = stats[from * kRows + row];
      part[r] = shares[from * share + k];
      m = fmaxf(m, s[r].x);
    }
    const float m0 = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int r = 0; r < kMaxSplits; ++r) {
      s[r].y += s[r].x - m0;
      mv = fmaxf(mv, s[r].y);
    }
    const float mv0 = mv == -INFINITY ? 0.f : mv;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < kMaxSplits; ++r)
      if (r < splits) {
        sum += s[r].z * fast_exp2(s[r].x - m0);
        add(acc, part[r], fast_exp2(s[r].y - mv0));
      }
    finish(row, i, m, mv, sum, acc);
  }
}

// What a block spends outside its tiles, in tiles of a warp (start, first loads, merge: some 14,000 cycles under
// load, against 3,200 for a tile).
constexpr double kOverhead = 4.5;

template <int DP, int HR, bool SPLIT, bool VEC>
int launch(Params p, int batch, cudaStream_t st) {
  const size_t smem = (size_t)kWarps * Layout<DP, HR>::kBytes + Layout<DP, HR>::kInbox;
  auto kernel = decode8_kernel<DP, HR, SPLIT, VEC>;
  if (smem > 48 * 1024) {
    static std::atomic<uint64_t> done{0};
    MSA_CUDA_RETURN(allow_smem(kernel, (int)smem, done));
  }
  static std::atomic<int> resident{0};  // blocks to an SM
  int per_sm = resident.load(std::memory_order_relaxed);
  if (per_sm == 0) {
    MSA_CUDA_RETURN(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kWarps * 32, smem));
    per_sm = std::max(per_sm, 1);
    resident.store(per_sm, std::memory_order_relaxed);
  }
  // Less than a wave of items: each on a cluster of the size that finishes first. More: a block to an item costs the
  // least in merging, but the blocks behind the last whole wave would run on a chip that is mostly idle. If they are
  // no more than half a wave, as many items, or a sixth of a wave if that is more, go to pairs of blocks, first: the
  // lone blocks behind them start at another time than the others, and the pairs' slots take the last ones. Measured
  // (16 blocks, 8 groups of 128; a wave is 444 items): 64 requests 61.7 us (70.4 with lone blocks alone, 69.6 with
  // clusters of 4, 62.1 with pairs for the 68 items over and above the wave alone), 56 requests 56.6 (57.6, 69.5,
  // 57.3), 128 requests 103.3 (110, 114, 103.8); 80 requests, 196 items behind the wave, 71.6 (80.7); 96, 324 items
  // behind it: 83.4 alone, 90.4 with pairs.
  const int64_t head_tiles = ceil_div(p.q_heads / p.groups, 16), items = (int64_t)batch * p.groups;
  const int64_t slots = std::max<int64_t>(148 * per_sm / head_tiles, 1), behind = items % slots;
  const int64_t tiles = (int64_t)p.topk * ((p.block + kTile - 1) / kTile);
  int64_t shared = 0;
  if (items < slots) {
    double best = 0;
    for (int shift = 0; (1 << shift) <= kMaxSplits; ++shift) {
      if (shift && ((int64_t)kWarps << (shift - 1)) >= tiles) break;  // no more warps than tiles
      const double waves = (double)(((items << shift) + slots - 1) / slots);
      const double cost = waves * ((double)tiles / (kWarps << shift) + kOverhead);
      if (shift == 0 || cost < best) best = cost, p.split_shift = shift, shared = shift ? items : 0;
    }
  } else if (behind > 0 && behind <= slots / 2 && tiles > kWarps) {
    p.split_shift = 1;
    shared = std::max(behind, slots / 6);
    shared += (items - shared) & 1;  // whole clusters of lone blocks
  }
  p.shared = (int)shared;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((shared << p.split_shift) + items - shared), (unsigned)head_tiles);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {1u << p.split_shift, 1, 1};
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
  p.by_page = FastDiv((uint32_t)page_size);
  p.uniform = page_size % 16 == 0 && block_size % 16 == 0;
  const bool vec = head_dim % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(out) % 16 == 0 && reinterpret_cast<uintptr_t>(k_cache) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(v_cache) % 16 == 0 &&
                   (k_page_stride | k_slot_stride | k_head_stride) % 16 == 0 &&
                   (v_page_stride | v_slot_stride | v_head_stride) % 16 == 0;
  cudaStream_t st = as_stream(stream);
  const bool few = q_heads / groups <= 8;
  if (head_dim <= 64) return few ? launch_dim<64, 1>(p, batch, vec, st) : launch_dim<64, 2>(p, batch, vec, st);
  if (head_dim <= 128) return few ? launch_dim<128, 1>(p, batch, vec, st) : launch_dim<128, 2>(p, batch, vec, st);
  return few ? launch_dim<256, 1>(p, batch, vec, st) : launch_dim<256, 2>(p, batch, vec, st);
}
