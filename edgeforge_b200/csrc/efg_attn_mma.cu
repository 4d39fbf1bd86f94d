// efg_attn_mma.cu - attention on the warp-level tensor cores, with the key axis split over warps and over a
// cluster: calls of few rows that the decode kernel does not take, chunks of up to 64 rows per key head, FP32
// heads above 64, scales of zero and below, wide groups, odd pages.
//
// Rows of one key head are packed: row i * group + h of a sequence is query head h of the group
// at its i-th new token, so a decode step's group of heads shares one pass over the keys. A CTA
// owns 16 rows (its four warps take a quarter of every 64-key tile) or 64 rows, or 128 (16 per
// warp), and a share of the tiles; keys and values arrive through a ring of cp.async stages. Softmax is the
// running maximum and sum in FP32; partial results (maximum, sum, weighted values) meet in shared
// memory, first across warps, then across the cluster, in rank order: no atomics, no workspace,
// no second launch, the same bits on every call.
//
// 16-bit types: mma m16n8k16, weights rounded to the type before the value product (the sum uses
// the unrounded weights). F32: every operand is split x = hi + lo into two 11-bit TF32 parts and
// a product is hi hi + hi lo + lo hi (m16n8k8): what is left out is below 2^-21 of |x y|, so the
// result keeps FP32 accuracy at a sixth of the 16-bit rate, still above the CUDA cores' FP32.
//
// What bounds it: in F32 the warp-level tensor cores and the splits beside them (2048 tokens, 32 query and 4 key
// heads of 128, FP32: 695 us, 49 TFLOP/s of the formula's products, 148 TFLOP/s of TF32 ones); of few rows the
// latency of a tile (two loads and two products in sequence). At head size 128 the F32 sums of 64 rows and more take
// the registers, so the queries wait in shared memory (1225 -> 1046 us) and eight warps share a tile (-> 695).
#include <algorithm>
#include <type_traits>

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "efg_attn.cuh"
#include "efg_attn_launch.h"
#include "efg_attn_warp.cuh"
#include "efg_host.h"

namespace cg = cooperative_groups;

namespace efg {
namespace {

constexpr int kKeys = 64;      // keys of a tile
constexpr int kMaxCluster = 16;
// Four warps, or one for every 16 rows of a larger tile.
constexpr int threads_of(int MT) { return MT > 4 ? 32 * MT : 128; }

template <typename T, int D>
constexpr int stage_bytes() {
  return 2 * kKeys * D * static_cast<int>(sizeof(T));
}
// Calls of few rows wait for their loads: about 96 KB are in flight in the stages of the CTAs that fit on an SM.
template <typename T, int D, int MT>
constexpr int stages() {
  return stage_bytes<T, D>() <= 16384 ? 4 : MT > 4 ? 2 : 3;
}
// Wide F32 queries of large tiles wait in shared memory: the registers are for sums.
template <typename T, int D, int MT>
constexpr bool query_in_smem = sizeof(T) == 4 && D == 128 && MT > 1;

// 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Where 16-byte chunk c of key row r lies: the chunks of a row are exchanged so that the eight
// addresses of every shared-memory phase fall into different banks. 16-bit: ldmatrix takes one
// chunk of 8 rows. F32 keys: a quad of lanes takes 4 chunks of one row, two rows a phase. F32
// values: a phase takes 2 chunks of the four rows 2t (or 2t + 1).
template <typename T>
__device__ __forceinline__ int key_chunk(int r, int c) {
  return sizeof(T) == 2 ? c ^ (r & 7) : c ^ ((r & 1) << 2);
}
template <typename T>
__device__ __forceinline__ int value_chunk(int r, int c) {
  return sizeof(T) == 2 ? c ^ (r & 7) : c ^ (((r >> 1) & 3) << 1);
}

template <typename T, int D, int MT>
__global__ void __launch_bounds__(threads_of(MT), (sizeof(T) == 4 && D == 128) ? 1 : 2)
    attn_mma_kernel(const AttnParams p, const int tiles_per_seq) {
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int kRows = 16 * MT, kRowBytes = D * static_cast<int>(sizeof(T)), kChunks = kRowBytes / 16;
  constexpr int kThreads = threads_of(MT), kWarps = kThreads / 32;
  constexpr int kStages = stages<T, D, MT>(), kTile = kKeys * kRowBytes;
  constexpr int NT = MT == 1 ? 2 : 8;  // 8-key column groups of a warp's scores
  constexpr int KK = D / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int32_t slot_s[2][kKeys];
  __shared__ int64_t scan_s[kWarps + 2];
  __shared__ float top_s[kWarps][16], sum_s[kWarps][16];  // per warp, then (row order) per CTA
  __shared__ float part_top[16 * kWarps], part_sum[16 * kWarps];
  __shared__ int redo_s[16 * kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  cg::cluster_group cluster = cg::this_cluster();
  const int splits = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int kvh = blockIdx.y;
  const int64_t tile_id = blockIdx.x / splits;

  pdl_wait();
  pdl_launch_dependents();
  if (tiles_per_seq == 0 && blockIdx.x == 0 && kvh == 0) check_offsets(p);
  RowTile rt;
  if (tiles_per_seq > 0) {
    rt.seq = tile_id / tiles_per_seq;
    rt.index = tile_id - rt.seq * tiles_per_seq;
  } else if (!find_tile<kThreads>(p, tile_id, p.group, kRows, scan_s, rt)) {
    return;  // uniform over the cluster
  }
  Chunk c;
  if (!chunk_of_seq(p, rt.seq, c)) return;
  const int64_t m = c.end - c.begin;
  const int64_t tiles_here = (m * p.group + kRows - 1) / kRows;
  if (rt.index >= tiles_here) return;
  const int64_t row0 = (tiles_here - 1 - rt.index) * kRows;  // packed rows of this tile: row0 .., the last tile first
  const int64_t rows_here = min(static_cast<int64_t>(kRows), m * p.group - row0);
  const int first_token = static_cast<int>(row0 / p.group), last_token = static_cast<int>((row0 + rows_here - 1) / p.group);
  const int see_first = seen_by(c, c.begin + first_token), see_all = seen_by(c, c.begin + last_token);
  const int tiles = static_cast<int>((see_all + kKeys - 1) / kKeys);
  const int tile_begin = static_cast<int>(static_cast<int64_t>(tiles) * rank / splits);
  const int tile_end = static_cast<int>(static_cast<int64_t>(tiles) * (rank + 1) / splits);

  // ---- this warp's rows
  const int wrow = MT == 1 ? 0 : warp * 16;
  int sees[2];  // rows g and g + 8 of the warp
  const T* qrow[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = wrow + g + 8 * i;
    if (r < rows_here) {
      const int64_t token = (row0 + r) / p.group;
      const int head = kvh * p.group + static_cast<int>(row0 + r - token * p.group);
      sees[i] = seen_by(c, c.begin + static_cast<int>(token));
      qrow[i] = static_cast<const T*>(p.q) + (c.begin + token) * p.q_stride + static_cast<int64_t>(head) * p.head_dim;
    } else {
      sees[i] = 0;
      qrow[i] = nullptr;
    }
  }

  // ---- key slots of a tile, one thread per key: looked up a tile ahead of its copies
  auto slot_of = [&](int tile) -> int32_t {
    const int j = tile * kKeys + tid;
    if (tile >= tile_end || j >= see_all) return -1;
    return static_cast<int32_t>(key_row(p, c, j));
  };
  const uint32_t base = smem_addr(smem);
  auto issue = [&](int tile, int buf) {
    const uint32_t ks = base + static_cast<uint32_t>(buf) * (2 * kTile), vs = ks + kTile;
    const int32_t* slots = slot_s[tile & 1];
    const int64_t head_off = static_cast<int64_t>(kvh) * p.head_dim;
#pragma unroll 4
    for (int e = tid; e < kKeys * kChunks; e += kThreads) {
      const int r = e / kChunks, ch = e % kChunks;
      const int64_t slot = slots[r];
      const bool ok = slot >= 0 && ch * (16 / static_cast<int>(sizeof(T))) < p.head_dim;
      const T* k = static_cast<const T*>(p.k) + (ok ? slot * p.k_stride + head_off + ch * (16 / sizeof(T)) : 0);
      const T* v = static_cast<const T*>(p.v) + (ok ? slot * p.v_stride + head_off + ch * (16 / sizeof(T)) : 0);
      cp_async16(ks + r * kRowBytes + key_chunk<T>(r, ch) * 16, k, ok);
      cp_async16(vs + r * kRowBytes + value_chunk<T>(r, ch) * 16, v, ok);
    }
  };
  // the first stages: slots of one tile at a time
  for (int s = 0; s < kStages - 1; ++s) {
    if (tid < kKeys) slot_s[(tile_begin + s) & 1][tid] = slot_of(tile_begin + s);
    __syncthreads();
    if (tile_begin + s < tile_end) issue(tile_begin + s, s);
    cp_async_commit();
  }
  if (tid < kKeys) slot_s[(tile_begin + kStages - 1) & 1][tid] = slot_of(tile_begin + kStages - 1);

  // ---- queries as A fragments (F32: the four dims 16 kk + 4 t .. + 3 of both rows)
  constexpr bool kQueryInSmem = query_in_smem<T, D, MT>;
  const uint32_t q_smem = base + kStages * 2 * kTile;
  uint32_t qa[kF32 ? 1 : KK][4];
  float4 qf[kF32 && !kQueryInSmem ? KK : 1][2];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    if constexpr (kF32) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int d = 16 * kk + 4 * t;
        const float4 v = qrow[i] && d < p.head_dim ? *reinterpret_cast<const float4*>(qrow[i] + d) : make_float4(0, 0, 0, 0);
        if constexpr (kQueryInSmem) {
          const int r = wrow + g + 8 * i;
          *reinterpret_cast<float4*>(smem + (q_smem - base) + r * kRowBytes + key_chunk<T>(r, 4 * kk + t) * 16) = v;
        } else {
          qf[kk][i] = v;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 16 * kk + 8 * (i >> 1) + 2 * t;
        qa[kk][i] = qrow[i & 1] && d < p.head_dim ? *reinterpret_cast<const uint32_t*>(qrow[i & 1] + d) : 0u;
      }
    }
  }

  const float scale2 = p.scale * 1.4426950408889634f;
  float acc[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};

  for (int tile = tile_begin; tile < tile_end; ++tile) {
    const int it = tile - tile_begin, buf = it % kStages;
    cp_async_wait<kStages - 2>();
    __syncthreads();  // this tile has landed; its predecessor's stage and slots are free
    if (tile + kStages - 1 < tile_end) issue(tile + kStages - 1, (it + kStages - 1) % kStages);
    cp_async_commit();
    const int32_t next_slot = tid < kKeys ? slot_of(tile + kStages) : -1;

    const uint32_t ks = base + static_cast<uint32_t>(buf) * (2 * kTile), vs = ks + kTile;
    const int key0 = MT == 1 ? warp * 16 : 0;
    // F32: the small products apart; under small tiles the large ones of 32 dims at a time, added to the score by an
    // FP32 addition: the matrix instructions cut off where those round, at every step of a chain.
    constexpr bool kSteps = kF32 && MT == 1;
    float s[NT][4], s2[kF32 ? NT : 1][4], far[kSteps ? NT : 1][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[n][i] = 0.f;
        if constexpr (kF32) s2[n][i] = 0.f;
        if constexpr (kSteps) far[n][i] = 0.f;
      }
    // ---- scores
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      if constexpr (kF32) {
        uint32_t qh[2][4], ql[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = wrow + g + 8 * i;  // (this lane's own stores, or registers)
          const float4 q =
              kQueryInSmem ? lds128(q_smem + r * kRowBytes + key_chunk<T>(r, 4 * kk + t) * 16) : qf[kQueryInSmem ? 0 : kk][i];
          split_tf32(q.x, qh[i][0], ql[i][0]);
          split_tf32(q.y, qh[i][1], ql[i][1]);
          split_tf32(q.z, qh[i][2], ql[i][2]);
          split_tf32(q.w, qh[i][3], ql[i][3]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int r = key0 + 8 * n + g;
          const float4 kv = lds128(ks + r * kRowBytes + key_chunk<T>(r, 4 * kk + t) * 16);
          uint32_t kh[4], kl[4];
          split_tf32(kv.x, kh[0], kl[0]);
          split_tf32(kv.y, kh[1], kl[1]);
          split_tf32(kv.z, kh[2], kl[2]);
          split_tf32(kv.w, kh[3], kl[3]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t ah[4] = {qh[0][2 * h], qh[1][2 * h], qh[0][2 * h + 1], qh[1][2 * h + 1]};
            const uint32_t al[4] = {ql[0][2 * h], ql[1][2 * h], ql[0][2 * h + 1], ql[1][2 * h + 1]};
            mma_tf32(s2[n], ah, kl[2 * h], kl[2 * h + 1]);
            mma_tf32(s2[n], al, kh[2 * h], kh[2 * h + 1]);
            mma_tf32(s[n], ah, kh[2 * h], kh[2 * h + 1]);
          }
          if (kSteps && kk % 2 == 1 && kk + 1 < KK) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              far[kSteps ? n : 0][e] += s[n][e];
              s[n][e] = 0.f;
            }
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          const int i = lane >> 3, r = key0 + 8 * n + (i >> 1) * 8 + (lane & 7);
          uint32_t b[4];
          ldmatrix4(ks + r * kRowBytes + key_chunk<T>(r, 2 * kk + (i & 1)) * 16, b);
          mma16<T>(s[n], qa[kk], b[0], b[1]);
          mma16<T>(s[n + 1], qa[kk], b[2], b[3]);
        }
      }
    }
    if constexpr (kF32) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = (kSteps ? far[kSteps ? n : 0][e] + s[n][e] : s[n][e]) + s2[n][e];
    }
    // ---- softmax of this tile (base 2), rows g and g + 8
    float back[2];
    const int j0 = tile * kKeys + key0;
    const bool edge = j0 + 8 * NT > see_first;  // some row does not see all of these keys
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int limit = sees[i] - j0;
      float mx = top[i];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = s[n][2 * i + e];
          x *= scale2;
          if (edge && 8 * n + 2 * t + e >= limit) x = -INFINITY;
          mx = fmaxf(mx, x);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
      const float ref = mx == -INFINITY ? 0.f : mx;  // nothing seen yet: all weights 0
      back[i] = ex2(top[i] - ref);
      top[i] = mx;
      float add = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = s[n][2 * i + e];
          x = ex2(x - ref);
          add += x;
        }
      sum[i] = sum[i] * back[i] + add;
      if constexpr (!kF32) {
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          acc[n][2 * i] *= back[i];
          acc[n][2 * i + 1] *= back[i];
        }
      }
    }
    // ---- weighted values
    if constexpr (kF32) {
      // The products of one tile are summed from zero and added to the running sums by FP32 additions: the matrix
      // instructions cut off instead of rounding, which over a long row would shrink it (by 1.3e-5 at 8192 keys).
#pragma unroll
      for (int dc = 0; dc < D / 32; ++dc) {  // column g of group (dc, i) is dim 32 dc + 4 g + i
        float big[4][4] = {}, small[4][4] = {};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t ph[4], pl[4];  // A fragment: k = t is key 2t, k = t + 4 key 2t + 1
          split_tf32(s[n][0], ph[0], pl[0]);
          split_tf32(s[n][2], ph[1], pl[1]);
          split_tf32(s[n][1], ph[2], pl[2]);
          split_tf32(s[n][3], ph[3], pl[3]);
          const int r = key0 + 8 * n + 2 * t;
          const float4 v0 = lds128(vs + r * kRowBytes + value_chunk<T>(r, 8 * dc + g) * 16);
          const float4 v1 = lds128(vs + (r + 1) * kRowBytes + value_chunk<T>(r + 1, 8 * dc + g) * 16);
          const float a0[4] = {v0.x, v0.y, v0.z, v0.w}, a1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t h0, l0, h1, l1;
            split_tf32(a0[i], h0, l0);
            split_tf32(a1[i], h1, l1);
            mma_tf32(small[i], ph, l0, l1);
            mma_tf32(small[i], pl, h0, h1);
            mma_tf32(big[i], ph, h0, h1);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[4 * dc + i][e] = fmaf(acc[4 * dc + i][e], back[e >> 1], big[i][e] + small[i][e]);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        const uint32_t pa[4] = {pack2<T>(s[n][0], s[n][1]), pack2<T>(s[n][2], s[n][3]),
                                pack2<T>(s[n + 1][0], s[n + 1][1]), pack2<T>(s[n + 1][2], s[n + 1][3])};
#pragma unroll
        for (int dd = 0; dd < D / 16; ++dd) {
          const int i = lane >> 3, r = key0 + 8 * n + (i & 1) * 8 + (lane & 7);
          uint32_t b[4];
          ldmatrix4_trans(vs + r * kRowBytes + value_chunk<T>(r, 2 * dd + (i >> 1)) * 16, b);
          mma16<T>(acc[2 * dd], pa, b[0], b[1]);
          mma16<T>(acc[2 * dd + 1], pa, b[2], b[3]);
        }
      }
    }
    if (tid < kKeys) slot_s[(tile + kStages) & 1][tid] = next_slot;
  }
  cp_async_wait<0>();
  __syncthreads();  // the stages become the exchange area

  // ---- partial results: [row][D] weighted values, maximum and sum per row
  float* o_s = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float v = sum[i];
    v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
    v += __shfl_xor_sync(0xFFFFFFFFu, v, 2);
    if (t == 0) {
      top_s[warp][g + 8 * i] = top[i];
      sum_s[warp][g + 8 * i] = v;
    }
    float* o = o_s + (warp * 16 + g + 8 * i) * D;
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = kF32 ? 32 * (n / 4) + 8 * t + 4 * e + n % 4 : 8 * n + 2 * t + e;
        o[d] = acc[n][2 * i + e];
      }
  }
  __syncthreads();
  if constexpr (MT == 1) {  // the four warps saw different keys of the same rows
    for (int e = tid; e < 16 * D; e += kThreads) {
      const int r = e / D;
      float mx = top_s[0][r];
#pragma unroll
      for (int w = 1; w < 4; ++w) mx = fmaxf(mx, top_s[w][r]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      float v = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = ex2(top_s[w][r] - ref);
        v += f * o_s[w * 16 * D + e];
        l += f * sum_s[w][r];
      }
      o_s[e] = v;
      if (e % D == 0) {
        part_top[r] = mx;
        part_sum[r] = l;
      }
    }
  } else if (tid < kRows) {
    part_top[tid] = top_s[tid >> 4][tid & 15];
    part_sum[tid] = sum_s[tid >> 4][tid & 15];
  }
  if (tid < kRows) redo_s[tid] = 0;
  if (splits > 1)
    cluster.sync();
  else
    __syncthreads();

  // ---- this CTA's share of the rows over all splits, in rank order
  const int share = (kRows + splits - 1) / splits, r_lo = rank * share;
  const int r_hi = min(static_cast<int>(rows_here), min(kRows, r_lo + share));
  for (int e = tid; e < max(0, r_hi - r_lo) * D; e += kThreads) {
    const int r = r_lo + e / D, d = e % D;
    float v, l;
    if (splits == 1) {
      v = o_s[r * D + d];
      l = part_sum[r];
    } else {
      float mx = -INFINITY;
      for (int w = 0; w < splits; ++w) mx = fmaxf(mx, cluster.map_shared_rank(part_top, w)[r]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      v = l = 0.f;
      for (int w = 0; w < splits; ++w) {
        const float f = ex2(cluster.map_shared_rank(part_top, w)[r] - ref);
        v += f * cluster.map_shared_rank(o_s, w)[r * D + d];
        l += f * cluster.map_shared_rank(part_sum, w)[r];
      }
    }
    if (d < p.head_dim) {
      const int64_t token = (row0 + r) / p.group;
      const int head = kvh * p.group + static_cast<int>(row0 + r - token * p.group);
      const float o = l == 0.f ? 0.f : v / l;
      if (!(fabsf(o) <= 3.402823466e38f)) redo_s[r] = 1;
      static_cast<T*>(p.out)[((c.begin + token) * p.heads + head) * p.head_dim + d] = attn_narrow<T>(o);
    }
  }
  if (see_first < see_all) {  // a row may not be reached by what lies at positions it does not see
    __syncthreads();
    for (int r = r_lo + warp; r < r_hi; r += kWarps) {
      if (!redo_s[r]) continue;
      const int64_t token = (row0 + r) / p.group;
      const int head = kvh * p.group + static_cast<int>(row0 + r - token * p.group);
      if (reached_from_behind<T>(p, c, c.begin + token, kvh, see_all))
        attend_row<T>(p, c, c.begin + token, head);
    }
  }
  if (splits > 1) cluster.sync();  // the peers read this CTA's shared memory until here
}

template <typename T, int D, int MT>
int launch(const AttnParams& p, int64_t tiles, int tiles_per_seq, int splits, cudaStream_t s) {
  const auto fn = attn_mma_kernel<T, D, MT>;
  const void* key = reinterpret_cast<const void*>(fn);
  const size_t smem = static_cast<size_t>(stages<T, D, MT>()) * stage_bytes<T, D>() +
                      (query_in_smem<T, D, MT> ? 16 * MT * D * sizeof(T) : 0);
  if (int st = ensure_smem_attr(key, smem)) return st;
  if (splits > 8)
    if (int st = ensure_wide_cluster(key)) return st;
  if (tiles * splits > 0x7FFFFFFFll) return fail(EFG_EINVAL, "attention: too many rows");
  cudaLaunchConfig_t cf{};
  cf.gridDim = dim3(static_cast<unsigned>(tiles * splits), static_cast<unsigned>(p.kv_heads));
  cf.blockDim = dim3(threads_of(MT));
  cf.dynamicSmemBytes = smem;
  cf.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(splits), 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cf.attrs = attr;
  cf.numAttrs = 2;
  EFG_TRY_CUDA(cudaLaunchKernelEx(&cf, fn, p, tiles_per_seq), "attention launch");
  return EFG_OK;
}

template <typename T, int D>
int dispatch(const AttnParams& p, int64_t max_rows, int64_t max_keys, int sms, cudaStream_t s) {
  const bool wide = sizeof(T) == 4 && D == 128;
  // Tiles of one sequence at fixed places when that launches no more of them than an upper bound
  // over the whole batch (a decode step: exactly one per sequence), else found by a scan.
  auto fixed = [&](int rows) { return p.n_seqs * ((max_rows + rows - 1) / rows); };
  auto bound = [&](int rows) { return p.n_rows * p.group / rows + p.n_seqs; };
  auto tiles_of = [&](int rows) { return std::min(fixed(rows), bound(rows)); };
  // 16 or 64 rows. Wide FP32 heads leave room for one CTA per SM, four warps: 128 rows on eight warps where 64-row
  // tiles would not all run at once (2048 tokens: 692 against 1046 us; 3 prompts of up to 214 tokens, 8 key heads,
  // 64-row tiles on 100 SMs: 58 against 48).
  const int rows = max_rows <= 16 ? 16 : wide && max_rows > 64 && tiles_of(64) * p.kv_heads > sms ? 128 : 64;
  const int64_t tiles = tiles_of(rows);
  const int per_seq = fixed(rows) <= bound(rows) ? static_cast<int>((max_rows + rows - 1) / rows) : 0;
  // Split the keys until there are about four CTAs per SM (one, where no more fit: 4 chunks of up to 169 FP32 tokens,
  // 4 key heads of 128: 48 against 89 us), but leave each two tiles of keys.
  const int64_t enough = (wide && rows > 16 ? 1 : 4) * sms;
  int splits = 1;
  while (splits < kMaxCluster && tiles * p.kv_heads * splits * 2 <= enough && max_keys >= kKeys * 4 * splits) splits *= 2;
  if (rows == 16) return launch<T, D, 1>(p, tiles, per_seq, splits, s);
  if constexpr (sizeof(T) == 4 && D == 128)
    if (rows == 128) return launch<T, D, 8>(p, tiles, per_seq, splits, s);
  return launch<T, D, 4>(p, tiles, per_seq, splits, s);
}

}  // namespace

bool attn_mma_takes(int type, const AttnParams& p) {
  const size_t es = type == EFG_F32 ? 4 : 2, unit = 16 / es;
  auto ok = [&](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  return p.head_dim <= 128 && p.head_dim % unit == 0 && p.q_stride % unit == 0 && p.k_stride % unit == 0 &&
         p.v_stride % unit == 0 && ok(p.q) && ok(p.k) && ok(p.v);
}

int launch_attn_mma(int type, const AttnParams& p, int sms, cudaStream_t s) {
  const int64_t max_keys = p.kv_len ? p.max_pages * p.page_size : p.n_rows;
  const int64_t max_rows = std::min(p.kv_len ? p.max_new : p.n_rows, p.n_rows) * p.group;
  if (type == EFG_F32)
    return p.head_dim <= 64 ? dispatch<float, 64>(p, max_rows, max_keys, sms, s)
                            : dispatch<float, 128>(p, max_rows, max_keys, sms, s);
  if (type == EFG_F16)
    return p.head_dim <= 64 ? dispatch<__half, 64>(p, max_rows, max_keys, sms, s)
                            : dispatch<__half, 128>(p, max_rows, max_keys, sms, s);
  return p.head_dim <= 64 ? dispatch<__nv_bfloat16, 64>(p, max_rows, max_keys, sms, s)
                          : dispatch<__nv_bfloat16, 128>(p, max_rows, max_keys, sms, s);
}

}  // namespace efg
