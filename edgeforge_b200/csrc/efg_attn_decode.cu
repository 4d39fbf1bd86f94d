// efg_attn_decode.cu - attention of at most 16 rows per key head (a decode step's head group, a few
// drafted tokens): bound by reading the keys and values once.
//
// The keys of a sequence are cut into parts of `chunk` positions; one CTA takes one part of one key
// head for all of its rows. A producer thread streams 64-key tiles (K, V) through a ring by TMA,
// page by page, and four consumer warps take 16 keys of every tile each, with their own running
// maximum and sum, so nothing but the ring's barriers is shared until the end. Partial rows of the
// warps meet in shared memory; with more than one part they go to the caller's workspace and a second
// launch (already resident by then: programmatic dependent launch) joins them in part order. The parts
// have the same size whatever the sequences' lengths are, so ragged batches stay balanced, and they
// may be any number, so one long sequence still fills every SM.
//
// Arithmetic as in efg_attn_mma.cu: 16-bit types by mma m16n8k16; F32 by TF32 parts. Up to 8 rows of
// F32 fill the 16 rows of the matrix instruction with both parts of the queries (rows 0-7 hi, 8-15 lo):
// two products (times K hi and K lo) instead of three, and lo lo comes with them. The same holds for
// the weights and the values.
//
// Shared memory tiles are TMA's 128-byte swizzle: 16-byte chunk c of row r lies at c ^ (r & 7). For F32 the
// lanes of a quad row g take key (g >> 1) + 4 (g & 1) of each 8, and chunk (g >> 1) + 4 (g & 1) of the values,
// which makes the eight addresses of every shared-memory phase fall into different banks.
#include <algorithm>

#include <cuda_runtime.h>

#include "efg_attn.cuh"
#include "efg_attn_launch.h"
#include "efg_attn_warp.cuh"
#include "efg_host.h"

namespace efg {
namespace {

constexpr int kConsumers = 4, kThreads = 32 * (kConsumers + 1);

template <typename T, int D>
struct Shape {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kKeys = kF32 && D == 128 ? 32 : 64;  // of a tile: 32 KB of K and V, 16 KB for small heads
  static constexpr int kPanels = D * static_cast<int>(sizeof(T)) / 128;
  static constexpr int kPanelBytes = kKeys * 128;
  static constexpr int kTileBytes = kPanels * kPanelBytes;  // K or V
  static constexpr int kStages = kTileBytes <= 8192 ? 4 : 2;  // 64 KB a CTA: three CTAs on an SM
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(kStages) * 2 * kTileBytes;
};

struct DecodeParams {
  AttnParams a;
  float* work;   // [seq][kv_head][part]{top[16], sum[16], o[16][D]}; null: one part each
  int chunk;     // positions of a part, a multiple of the tile
  int parts;     // parts that the grid has for every sequence
  int box_rows;  // rows of one TMA box
};

// The rows of one sequence under one key head.
struct Rows {
  Chunk c;
  int rows;                     // packed rows: token * group + head
  int64_t see_first, see_all;   // keys that the first and the last token see
};

__device__ __forceinline__ bool rows_of(const AttnParams& p, int64_t seq, Rows& w) {
  if (!chunk_of_seq(p, seq, w.c)) return false;
  const int64_t m = w.c.end - w.c.begin;
  if (m == 0 || m * p.group > kDecodeRows) return false;
  w.rows = static_cast<int>(m) * p.group;
  w.see_first = visible_keys(w.c.begin, w.c.begin, w.c.end, w.c.kv_len);
  w.see_all = visible_keys(w.c.end - 1, w.c.begin, w.c.end, w.c.kv_len);
  return true;
}

// Output element d.. of row r; true when it is not finite.
template <typename T>
__device__ __forceinline__ bool store_row(const AttnParams& p, const Rows& w, int kvh, int r, int d, float v, float l) {
  const int token = r / p.group;
  const float o = l == 0.f ? 0.f : v / l;
  static_cast<T*>(p.out)[((w.c.begin + token) * p.heads + kvh * p.group + r - token * p.group) * p.head_dim + d] =
      attn_narrow<T>(o);
  return !(fabsf(o) <= 3.402823466e38f);
}

// Rows marked in `redo` once more, alone, where something behind their last position reached them.
template <typename T>
__device__ __forceinline__ void redo_rows(const AttnParams& p, const Rows& w, int kvh, const int* redo, float* scratch,
                                          int warps) {
  if (w.see_first == w.see_all) return;  // every row sees every key that was used
  for (int r = threadIdx.x >> 5; r < w.rows; r += warps) {
    if (!redo[r]) continue;
    const int token = r / p.group;
    if (reached_from_behind<T>(p, w.c, w.c.begin + token, kvh, w.see_all))
      attend_row<T>(p, w.c, w.c.begin + token, kvh * p.group + r - token * p.group, scratch + (threadIdx.x >> 5) * 256);
  }
}

template <typename T, int D, bool kStack>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 && (D == 128 || !kStack) ? 2 : 3)
    attn_decode_kernel(const __grid_constant__ DecodeParams dp, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v) {
  using S = Shape<T, D>;
  constexpr bool kF32 = S::kF32;
  constexpr int kKeys = S::kKeys, kWarpKeys = kKeys / kConsumers, NT = kWarpKeys / 8, KK = D / 16;
  constexpr int kHalves = kStack ? 1 : 2;  // rows g (and g + 8) of a quad
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[S::kStages], empty[S::kStages];
  __shared__ float top_s[kConsumers][16], sum_s[kConsumers][16];
  __shared__ int redo_s[16];
  const AttnParams& p = dp.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int64_t seq = blockIdx.x / dp.parts;
  const int part = static_cast<int>(blockIdx.x - seq * dp.parts), kvh = blockIdx.y;
  pdl_launch_dependents();
  Rows w;
  if (!rows_of(p, seq, w)) return;
  const int64_t part_begin = static_cast<int64_t>(part) * dp.chunk;
  if (part > 0 && part_begin >= w.see_all) return;
  const int tile_begin = static_cast<int>(part_begin / kKeys);
  const int tile_end = static_cast<int>((min(w.see_all, part_begin + dp.chunk) + kKeys - 1) / kKeys);
  const uint32_t raw = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* ring = smem_raw + (base - raw);

  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kConsumers);
    }
    fence_barrier_init();
  }
  if (tid < 16) redo_s[tid] = 0;
  __syncthreads();

  float acc[D / 8][4];
  float top[kHalves], sum[kHalves];
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
#pragma unroll
  for (int i = 0; i < kHalves; ++i) top[i] = -INFINITY, sum[i] = 0.f;

  if (warp == kConsumers) {
    // ---- producer: a lane per box of a tile (page by page), K and V
    const int boxes = kKeys / dp.box_rows, b = lane % boxes, panel = lane / boxes;
    auto row_of = [&](int tile) -> int32_t {
      const int64_t pos = static_cast<int64_t>(tile) * kKeys + b * dp.box_rows;
      if (tile >= tile_end) return 0;
      if (!p.kv_len) return static_cast<int32_t>(w.c.begin + pos);
      const int64_t row = pos < w.see_all ? key_row(p, w.c, pos) : -1;
      return static_cast<int32_t>(row >= 0 ? row : p.n_pages * p.page_size);  // outside: zeros
    };
    int32_t row = row_of(tile_begin);
    bool ok = true;
    int issued = 0;
    for (int tile = tile_begin; tile < tile_end; ++tile) {
      const int it = tile - tile_begin, st = it % S::kStages;
      const int32_t next = row_of(tile + 1);
      if (it >= S::kStages) ok = wait_own(&empty[st], ((it / S::kStages) - 1) & 1, p.err);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&full[st], 2 * S::kTileBytes);
      __syncwarp();
      uint8_t* dst = ring + st * 2 * S::kTileBytes + b * dp.box_rows * 128;
      for (int h = panel; h < S::kPanels; h += 32 / boxes) {
        constexpr int kPerPanel = 128 / static_cast<int>(sizeof(T));
        tma_load_3d(dst + h * S::kPanelBytes, &map_k, kPerPanel * h, kvh, row, &full[st]);
        tma_load_3d(dst + S::kTileBytes + h * S::kPanelBytes, &map_v, kPerPanel * h, kvh, row, &full[st]);
      }
      ++issued;
      row = next;
    }
    if (!ok)  // the copies in flight land before the shared memory is given back
      for (int it = max(0, issued - S::kStages); it < issued; ++it)
        wait_own(&full[it % S::kStages], (it / S::kStages) & 1, p.err);
  } else {
    // ---- queries as A fragments
    const T* qrow[2];
    int64_t sees[kHalves];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = kStack ? g : g + 8 * i;
      const int token = r / p.group;
      const bool live = r < w.rows;
      qrow[i] = live ? static_cast<const T*>(p.q) + (w.c.begin + token) * p.q_stride +
                           static_cast<int64_t>(kvh * p.group + r - token * p.group) * p.head_dim
                     : nullptr;
      if (i < kHalves) sees[i] = live ? visible_keys(w.c.begin + token, w.c.begin, w.c.end, w.c.kv_len) : 0;
    }
    uint32_t qa[kF32 ? 1 : KK][4], qs[kStack ? KK : 1][2][4];
    float4 qf[kF32 && !kStack ? KK : 1][2];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      if constexpr (kF32) {
        const int d = 16 * kk + 4 * t;
        const float4 zero = make_float4(0, 0, 0, 0);
        if constexpr (kStack) {
          const float4 q = qrow[0] && d < p.head_dim ? *reinterpret_cast<const float4*>(qrow[0] + d) : zero;
          // step h: k = t is component 2h, k = t + 4 component 2h + 1; rows g hi, g + 8 lo
          split_tf32(q.x, qs[kk][0][0], qs[kk][0][1]);
          split_tf32(q.y, qs[kk][0][2], qs[kk][0][3]);
          split_tf32(q.z, qs[kk][1][0], qs[kk][1][1]);
          split_tf32(q.w, qs[kk][1][2], qs[kk][1][3]);
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            qf[kk][i] = qrow[i] && d < p.head_dim ? *reinterpret_cast<const float4*>(qrow[i] + d) : zero;
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
    const int key0 = warp * kWarpKeys, perm = (g >> 1) + 4 * (g & 1);
    bool ok = true;

    for (int tile = tile_begin; tile < tile_end; ++tile) {
      const int it = tile - tile_begin, st = it % S::kStages;
      ok = wait_own(&full[st], (it / S::kStages) & 1, p.err);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      const uint32_t ks = base + static_cast<uint32_t>(st) * (2 * S::kTileBytes), vs = ks + S::kTileBytes;
      const int64_t j0 = static_cast<int64_t>(tile) * kKeys + key0;
      if (j0 + kWarpKeys > w.see_all) {
        // values behind the last position become zeros: 0 times what may lie there need not be 0
        const int keep = static_cast<int>(max(int64_t{0}, w.see_all - j0));
        for (int e = lane; e < (kWarpKeys - keep) * S::kPanels * 8; e += 32) {
          const int r = key0 + keep + e / (S::kPanels * 8), h = (e / 8) % S::kPanels;
          *reinterpret_cast<uint4*>(ring + (vs - base) + h * S::kPanelBytes + r * 128 + (e % 8) * 16) =
              make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }
      float s[NT][4], s2[kStack ? NT : 1][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[n][i] = 0.f;
          if constexpr (kStack) s2[n][i] = 0.f;
        }
      // ---- scores
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if constexpr (kF32) {
          uint32_t qh[2][4], ql[2][4];
          if constexpr (!kStack) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              split_tf32(qf[kk][i].x, qh[i][0], ql[i][0]);
              split_tf32(qf[kk][i].y, qh[i][1], ql[i][1]);
              split_tf32(qf[kk][i].z, qh[i][2], ql[i][2]);
              split_tf32(qf[kk][i].w, qh[i][3], ql[i][3]);
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int r = key0 + 8 * n + perm;
            const float4 kv = lds128(ks + (kk >> 1) * S::kPanelBytes + r * 128 + (((4 * (kk & 1) + t) ^ (r & 7)) << 4));
            uint32_t kh[4], kl[4];
            split_tf32(kv.x, kh[0], kl[0]);
            split_tf32(kv.y, kh[1], kl[1]);
            split_tf32(kv.z, kh[2], kl[2]);
            split_tf32(kv.w, kh[3], kl[3]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if constexpr (kStack) {
                mma_tf32(s2[n], qs[kk][h], kl[2 * h], kl[2 * h + 1]);
                mma_tf32(s[n], qs[kk][h], kh[2 * h], kh[2 * h + 1]);
              } else {
                const uint32_t ah[4] = {qh[0][2 * h], qh[1][2 * h], qh[0][2 * h + 1], qh[1][2 * h + 1]};
                const uint32_t al[4] = {ql[0][2 * h], ql[1][2 * h], ql[0][2 * h + 1], ql[1][2 * h + 1]};
                mma_tf32(s[n], ah, kl[2 * h], kl[2 * h + 1]);
                mma_tf32(s[n], al, kh[2 * h], kh[2 * h + 1]);
                mma_tf32(s[n], ah, kh[2 * h], kh[2 * h + 1]);
              }
            }
          }
        } else {
#pragma unroll
          for (int n = 0; n < NT; n += 2) {
            const int i = lane >> 3, r = key0 + 8 * n + (i >> 1) * 8 + (lane & 7);
            uint32_t b[4];
            ldmatrix4(ks + (kk >> 2) * S::kPanelBytes + r * 128 + (((2 * (kk & 3) + (i & 1)) ^ (r & 7)) << 4), b);
            mma16<T>(s[n], qa[kk], b[0], b[1]);
            mma16<T>(s[n + 1], qa[kk], b[2], b[3]);
          }
        }
      }
      if constexpr (kStack) {  // both parts of the queries, both parts of the keys
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) s[n][e] = (s[n][e] + (s[n][e + 2] + s2[n][e])) + s2[n][e + 2];
      }
      // ---- softmax (base 2)
      const bool edge = j0 + kWarpKeys > w.see_first;
#pragma unroll
      for (int i = 0; i < kHalves; ++i) {
        const int limit = static_cast<int>(max(int64_t{0}, min(static_cast<int64_t>(kWarpKeys), sees[i] - j0)));
        float mx = top[i];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = s[n][2 * i + e];
            const int key = 8 * n + (kF32 ? t + 4 * e : 2 * t + e);
            x *= scale2;
            if (edge && key >= limit) x = -INFINITY;
            mx = fmaxf(mx, x);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
        const float ref = mx == -INFINITY ? 0.f : mx;
        const float back = ex2(top[i] - ref);
        const bool moved = mx != top[i];
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
        sum[i] = sum[i] * back + add;
        if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            acc[n][2 * i] *= back;
            acc[n][2 * i + 1] *= back;
            if constexpr (kStack) {
              acc[n][2] *= back;
              acc[n][3] *= back;
            }
          }
        }
      }
      // ---- weighted values
      if constexpr (kF32) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t ph[4], pl[4];  // A fragment: k = t is key t, k = t + 4 key t + 4 of the eight
          if constexpr (kStack) {
            split_tf32(s[n][0], ph[0], ph[1]);
            split_tf32(s[n][1], ph[2], ph[3]);
          } else {
            split_tf32(s[n][0], ph[0], pl[0]);
            split_tf32(s[n][2], ph[1], pl[1]);
            split_tf32(s[n][1], ph[2], pl[2]);
            split_tf32(s[n][3], ph[3], pl[3]);
          }
          const int r = key0 + 8 * n + t;  // and r + 4
#pragma unroll
          for (int dc = 0; dc < D / 32; ++dc) {  // column g of group (dc, i) is dim 32 dc + 4 perm + i
            const uint32_t panel = vs + dc * S::kPanelBytes;
            const float4 v0 = lds128(panel + r * 128 + ((perm ^ (r & 7)) << 4));
            const float4 v1 = lds128(panel + (r + 4) * 128 + ((perm ^ ((r + 4) & 7)) << 4));
            const float a0[4] = {v0.x, v0.y, v0.z, v0.w}, a1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t h0, l0, h1, l1;
              split_tf32(a0[i], h0, l0);
              split_tf32(a1[i], h1, l1);
              mma_tf32(acc[4 * dc + i], ph, l0, l1);
              if constexpr (!kStack) mma_tf32(acc[4 * dc + i], pl, h0, h1);
              mma_tf32(acc[4 * dc + i], ph, h0, h1);
            }
          }
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
            ldmatrix4_trans(vs + (dd >> 2) * S::kPanelBytes + r * 128 + (((2 * (dd & 3) + (i >> 1)) ^ (r & 7)) << 4), b);
            mma16<T>(acc[2 * dd], pa, b[0], b[1]);
            mma16<T>(acc[2 * dd + 1], pa, b[2], b[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
  }
  __syncthreads();  // the ring becomes the exchange area: [warp][16][D]

  float* o_s = reinterpret_cast<float*>(ring);
  if (warp < kConsumers) {
#pragma unroll
    for (int i = 0; i < kHalves; ++i) {
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
          const int d = kF32 ? 32 * (n / 4) + 4 * t + 16 * e + n % 4 : 8 * n + 2 * t + e;
          o[d] = kStack ? acc[n][e] + acc[n][e + 2] : acc[n][2 * i + e];
        }
    }
  }
  __syncthreads();
  const bool joined = dp.work && w.see_all > dp.chunk;  // more than one part: the second launch joins them
  float* slot = joined ? dp.work + ((seq * p.kv_heads + kvh) * dp.parts + part) * (16 * (D + 2)) : nullptr;
  for (int e = tid; e < w.rows * D; e += kThreads) {
    const int r = e / D, d = e % D;
    float mx = top_s[0][r];
#pragma unroll
    for (int x = 1; x < kConsumers; ++x) mx = fmaxf(mx, top_s[x][r]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float v = 0.f, l = 0.f;
#pragma unroll
    for (int x = 0; x < kConsumers; ++x) {
      const float f = ex2(top_s[x][r] - ref);
      v += f * o_s[(x * 16 + r) * D + d];
      l += f * sum_s[x][r];
    }
    if (joined) {
      slot[32 + e] = v;
      if (d == 0) {
        slot[r] = mx;
        slot[16 + r] = l;
      }
    } else if (d < p.head_dim) {
      if (store_row<T>(p, w, kvh, r, d, v, l)) redo_s[r] = 1;
    }
  }
  if (!joined) {
    __syncthreads();
    redo_rows<T>(p, w, kvh, redo_s, o_s, kThreads / 32);
  }
}

// Joins the parts of one sequence and key head: out = sum_x 2^(top_x - top) o_x / sum_x 2^(top_x - top) l_x.
template <typename T, int D>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ DecodeParams dp) {
  __shared__ float scratch[4 * 256];
  __shared__ int redo_s[16];
  const AttnParams& p = dp.a;
  const int64_t seq = blockIdx.x;
  const int kvh = blockIdx.y;
  if (threadIdx.x < 16) redo_s[threadIdx.x] = 0;
  __syncthreads();
  pdl_wait();
  Rows w;
  if (!rows_of(p, seq, w) || w.see_all <= dp.chunk) return;
  const int parts = static_cast<int>((w.see_all + dp.chunk - 1) / dp.chunk);
  const float* slots = dp.work + (seq * p.kv_heads + kvh) * dp.parts * static_cast<int64_t>(16 * (D + 2));
  const int r0 = blockIdx.z * 4, r = r0 + (threadIdx.x >> 5), lane = threadIdx.x & 31;  // one warp per row
  if (r < w.rows) {
    float mx = -INFINITY;
    for (int x = lane; x < parts; x += 32) mx = fmaxf(mx, slots[static_cast<int64_t>(x) * (16 * (D + 2)) + r]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
    const float ref = mx == -INFINITY ? 0.f : mx;
    float l = 0.f, acc[D / 32] = {};
    for (int x0 = 0; x0 < parts; x0 += 32) {  // weights of 32 parts at once, then their values in order
      const float* mine = slots + static_cast<int64_t>(x0 + lane) * (16 * (D + 2));
      const float f = x0 + lane < parts ? ex2(mine[r] - ref) : 0.f;
      const float fl = x0 + lane < parts ? f * mine[16 + r] : 0.f;
      const int n = min(32, parts - x0);
#pragma unroll 4
      for (int x = 0; x < n; ++x) {
        const float* o = slots + static_cast<int64_t>(x0 + x) * (16 * (D + 2)) + 32 + r * D;
        const float fx = __shfl_sync(0xFFFFFFFFu, f, x);
        l += __shfl_sync(0xFFFFFFFFu, fl, x);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] += fx * o[lane + 32 * i];
      }
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      if (lane + 32 * i < p.head_dim && store_row<T>(p, w, kvh, r, lane + 32 * i, acc[i], l)) redo_s[r] = 1;
  }
  __syncwarp();
  if (r < w.rows && redo_s[r] && w.see_first < w.see_all) {
    const int token = r / p.group;
    if (reached_from_behind<T>(p, w.c, w.c.begin + token, kvh, w.see_all))
      attend_row<T>(p, w.c, w.c.begin + token, kvh * p.group + r - token * p.group, scratch + (threadIdx.x >> 5) * 256);
  }
}

// How a call is cut: positions of a part and parts per sequence.
struct Cut {
  int chunk, parts;
};
Cut cut_of(int type, const AttnParams& p, int sms) {
  const int es = type == EFG_F32 ? 4 : 2, D = p.head_dim <= 64 ? 64 : 128;
  const int64_t max_keys = std::max<int64_t>(1, p.kv_len ? p.max_pages * p.page_size : p.n_rows);
  // Three CTAs on every SM when all sequences are as long as the table allows; but not below 128 positions
  // (a CTA's start and end cost as much as that) and not above 512 KB, which keeps ragged batches balanced.
  const int64_t even = (max_keys * p.n_seqs * p.kv_heads + 3 * sms - 1) / (3 * sms);
  const int64_t chunk = (std::max<int64_t>(128, std::min<int64_t>(even, (512 << 10) / (2 * D * es))) + 63) / 64 * 64;
  return Cut{static_cast<int>(chunk), static_cast<int>((max_keys + chunk - 1) / chunk)};
}

template <typename T, int D, bool kStack>
int launch(const DecodeParams& dp, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t s) {
  using S = Shape<T, D>;
  const auto fn = attn_decode_kernel<T, D, kStack>;
  if (int st = ensure_smem_attr(reinterpret_cast<const void*>(fn), S::kSmem)) return st;
  const AttnParams& p = dp.a;
  if (p.n_seqs * dp.parts > 0x7FFFFFFFll) return fail(EFG_EINVAL, "attention: too many rows");
  fn<<<dim3(static_cast<unsigned>(p.n_seqs * dp.parts), static_cast<unsigned>(p.kv_heads)), kThreads, S::kSmem, s>>>(
      dp, mk, mv);
  EFG_TRY_CUDA(cudaGetLastError(), "attention launch");
  if (!dp.work) return EFG_OK;
  cudaLaunchConfig_t cf{};
  const int64_t rows = std::min<int64_t>(kDecodeRows, std::min(p.kv_len ? p.max_new : p.n_rows, p.n_rows) * p.group);
  cf.gridDim = dim3(static_cast<unsigned>(p.n_seqs), static_cast<unsigned>(p.kv_heads),
                    static_cast<unsigned>((rows + 3) / 4));
  cf.blockDim = dim3(128);
  cf.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cf.attrs = attr;
  cf.numAttrs = 1;
  EFG_TRY_CUDA(cudaLaunchKernelEx(&cf, attn_join_kernel<T, D>, dp), "attention launch");
  return EFG_OK;
}

template <typename T, int D>
int dispatch(int type, const AttnParams& p, const Cut& cut, void* work, cudaStream_t s) {
  using S = Shape<T, D>;
  DecodeParams dp;
  dp.a = p;
  dp.work = cut.parts > 1 ? static_cast<float*>(work) : nullptr;
  dp.chunk = cut.chunk;
  dp.parts = cut.parts;
  dp.box_rows = p.kv_len ? static_cast<int>(std::min<int64_t>(p.page_size, S::kKeys)) : S::kKeys;
  const int64_t kv_rows = p.kv_len ? p.n_pages * p.page_size : p.n_rows;
  CUtensorMap mk, mv;
  if (!encode_heads_map(&mk, type, p.k, p.head_dim, p.kv_heads, kv_rows, p.k_stride, 1, dp.box_rows) ||
      !encode_heads_map(&mv, type, p.v, p.head_dim, p.kv_heads, kv_rows, p.v_stride, 1, dp.box_rows))
    return fail(EFG_ECUDA, "attention: the driver rejects a tensor map");
  if constexpr (S::kF32) {
    if (std::min(p.kv_len ? p.max_new : p.n_rows, p.n_rows) * p.group <= 8) return launch<T, D, true>(dp, mk, mv, s);
  }
  return launch<T, D, false>(dp, mk, mv, s);
}

}  // namespace

bool attn_decode_takes(int type, const AttnParams& p) {
  if (p.k_stride == 0 || p.v_stride == 0) return false;
  if (p.kv_len && (p.n_pages == 0 || p.page_size < 8 || (p.page_size & (p.page_size - 1)))) return false;
  const int64_t max_new = std::min(p.kv_len ? p.max_new : p.n_rows, p.n_rows);
  return attn_mma_takes(type, p) && max_new * p.group <= kDecodeRows;
}

size_t attn_decode_workspace(int type, const AttnParams& p, int sms) {
  const Cut cut = cut_of(type, p, sms);
  if (cut.parts <= 1) return 0;
  return static_cast<size_t>(p.n_seqs) * p.kv_heads * cut.parts * 16 * ((p.head_dim <= 64 ? 64 : 128) + 2) * sizeof(float);
}

int launch_attn_decode(int type, const AttnParams& p, int sms, void* work, cudaStream_t s) {
  const Cut cut = cut_of(type, p, sms);
  const bool small = p.head_dim <= 64;
  if (type == EFG_F32)
    return small ? dispatch<float, 64>(type, p, cut, work, s) : dispatch<float, 128>(type, p, cut, work, s);
  if (type == EFG_F16)
    return small ? dispatch<__half, 64>(type, p, cut, work, s) : dispatch<__half, 128>(type, p, cut, work, s);
  return small ? dispatch<__nv_bfloat16, 64>(type, p, cut, work, s) : dispatch<__nv_bfloat16, 128>(type, p, cut, work, s);
}

}  // namespace efg
