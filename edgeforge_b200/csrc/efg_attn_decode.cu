// efg_attn_decode.cu - attention of at most 16 rows per key head (a decode step's head group, a few
// drafted tokens): bound by reading the keys and values once. Measured: one BF16 row over 131072 positions,
// 8 key heads of 128, 88-91 us, 5.9-6.1 TB/s; 64 FP32 rows over up to 4000 positions, 4 key heads of 64, 45 us, 4.1 TB/s,
// where the TF32 splits take 42 % of the issue slots.
//
// The key tiles (64 positions) of all sequences and key heads form one line (each key head weighs its
// tiles and what its begin and end cost), which is cut into as many equal runs as there are CTAs resident
// on the GPU: whatever the lengths are, every SM gets the same bytes, and one long sequence fills the GPU as
// well as a large ragged batch (keys split over clusters, as in efg_attn_mma.cu: 102 us for the 64 rows). A producer warp streams
// a run's tiles (K, V) through a ring by TMA, page by page, across the borders of sequences; four
// consumer warps take 16 keys of every tile each, with their own running maximum and sum, so nothing
// but the ring's barriers is shared until a key head's part of the run ends. Then the warps' rows meet
// in shared memory. A key head that lies inside one run is written out; the pieces of one that is cut
// go to the caller's workspace (at most two per CTA) and a second launch, which is resident by then
// (programmatic dependent launch), joins them in order: no atomics, the same bits on every call.
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
#include "efg_tcgen05.cuh"

namespace efg {
namespace {

constexpr int kConsumers = 4, kThreads = 32 * (kConsumers + 1);
// What the begin and end of a key head cost, in key tiles: 200 BF16 rows over 50 to 4000 positions, 8 key heads of
// 128, 270 us (with a cost of 1: 302, of 4: 274). The weight of a run, at least: 16 rows over 8000 positions 94 us (of 1:
// 93, of 6: 98), 512 rows over 300 positions 145 (147, 153).
constexpr int kHeadCost = 2, kMinRun = 3;
constexpr int kMaxCtas = 1024;

template <typename T, int D>
struct Shape {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kKeys = kF32 && D == 128 ? 32 : 64;  // of a tile: 32 KB of K and V, 16 KB for small heads
  static constexpr int kPanels = D * static_cast<int>(sizeof(T)) / 128;
  static constexpr int kPanelBytes = kKeys * 128;
  static constexpr int kTileBytes = kPanels * kPanelBytes;  // K or V
  // about 64 KB of tiles in flight a CTA, three CTAs on an SM (two for wide heads)
  static constexpr int kCtas = D == 128 ? 2 : 3;
  static constexpr int kStages = kTileBytes <= 8192 ? 3 : 2;
  static constexpr size_t smem(int rows) {  // tiles, then every warp's rows in FP32
    return 1024 + static_cast<size_t>(kStages) * 2 * kTileBytes + static_cast<size_t>(kConsumers) * rows * D * 4;
  }
};

// A cut key head's pieces are slot `first` of CTA i (1: the last part of its run, 0: all of it) and
// slot 0 of the CTAs behind it.
struct alignas(16) JoinDesc {
  int32_t seq, kvh, first, parts;  // parts 0: nothing begins here that is cut
  int32_t begin, end, kv_len, pad;  // the sequence's chunk
};

struct DecodeParams {
  AttnParams a;
  JoinDesc* desc;  // [ctas]
  float* slots;    // [ctas][2]{top[16], sum[16], o[16][D]}; null: key heads are never cut
  int box_rows;    // rows of one TMA box
};

// The rows of one sequence under one key head.
struct Rows {
  Chunk c;
  int rows;                     // packed rows: token * group + head
  int see_first, see_all;       // keys that the first and the last token see
};

__device__ __forceinline__ bool rows_of(const AttnParams& p, int64_t seq, Rows& w) {
  if (!chunk_of_seq(p, seq, w.c)) return false;
  const int m = w.c.end - w.c.begin;
  if (m == 0 || m > kDecodeRows || m * p.group > kDecodeRows) return false;
  w.rows = m * p.group;
  w.see_first = seen_by(w.c, w.c.begin);
  w.see_all = seen_by(w.c, w.c.end - 1);
  return true;
}

// Output element d.. of row r; true when it is not finite.
template <typename T>
__device__ __forceinline__ bool store_row(const AttnParams& p, const Rows& w, int kvh, int r, int d, float v, float l) {
  const int token = r / p.group;
  const float o = l == 0.f ? 0.f : v / l;
  static_cast<T*>(p.out)[(static_cast<int64_t>(w.c.begin + token) * p.heads + kvh * p.group + r - token * p.group) * p.head_dim + d] =
      attn_narrow<T>(o);
  return !(fabsf(o) <= 3.402823466e38f);
}

// Rows marked in `redo` once more, alone, where something behind their last position reached them.
// One warp.
template <typename T>
__device__ __forceinline__ void redo_rows(const AttnParams& p, const Rows& w, int kvh, const int* redo, uint64_t* until = nullptr) {
  for (int r = 0; r < w.rows; ++r) {
    const int token = r / p.group;
    if (redo[r] && seen_by(w.c, w.c.begin + token) < w.see_all &&
        reached_from_behind<T>(p, w.c, w.c.begin + token, kvh, w.see_all))
      attend_row<T>(p, w.c, w.c.begin + token, kvh * p.group + r - token * p.group, until);
  }
}

// Place of dim d in a warp's row r of the exchange area: pieces of a row exchanged so that a fragment's
// eight rows fall into different banks (F32: 16-byte pieces, otherwise 8-byte ones).
template <bool kF32>
__device__ __forceinline__ int slab_at(int r, int d) {
  return kF32 ? (((d >> 2) ^ ((r & 1) << 2)) << 2) | (d & 3) : (((d >> 1) ^ ((r & 3) << 2)) << 1) | (d & 1);
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}

// The consumer warps alone.
__device__ __forceinline__ void consumer_barrier() {
  __syncwarp();
  asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumers) : "memory");
}

// Key tiles of a key head; one that sees nothing has one (its rows are zeros).
template <typename T, int D>
__device__ __forceinline__ int tiles_of(const Rows& w) {
  return max(1, (w.see_all + Shape<T, D>::kKeys - 1) / Shape<T, D>::kKeys);
}

// Weight of a sequence on the line: of each key head its begin and end, then its tiles; 1 per key head when
// they are never cut. 0 without new tokens.
template <typename T, int D>
__device__ __forceinline__ int weight_of(const DecodeParams& dp, int64_t seq) {
  Rows w;
  if (!rows_of(dp.a, seq, w)) return 0;
  return (dp.slots ? kHeadCost + tiles_of<T, D>(w) : 1) * dp.a.kv_heads;
}

// Walks the parts of a run: for each, the sequence, the key head and the tiles [from, to) of it.
template <typename T, int D>
struct Walk {
  int left, at;  // what is left of the run, and the place inside the sequence's weight
  int seq, kvh, from, to, all;
  Rows w;
  bool loaded;
  __device__ __forceinline__ void start(int s, int place, int count) {
    seq = s;
    at = place;
    left = count;
    loaded = false;
  }
  __device__ __forceinline__ bool next(const DecodeParams& dp) {
    const bool cut = dp.slots != nullptr;
    while (left > 0) {
      if (!loaded) {
        if (seq >= dp.a.n_seqs) return false;  // not reached: runs end with the line
        loaded = rows_of(dp.a, seq, w);
        if (loaded) all = tiles_of<T, D>(w);
      }
      const int weight = cut ? kHeadCost + all : 1;
      if (!loaded || at >= weight * dp.a.kv_heads) {
        ++seq;
        at = 0;
        loaded = false;
        continue;
      }
      kvh = at / weight;
      const int off = at - kvh * weight, step = min(weight - off, left);
      left -= step;
      at += step;
      from = cut ? max(0, off - kHeadCost) : 0;
      to = cut ? off + step - kHeadCost : all;
      if (to > from) return true;  // else the run ends before the head's first tile
    }
    return false;
  }
};

template <typename T, int D, bool kStack>
__global__ void __launch_bounds__(kThreads, Shape<T, D>::kF32 && !kStack ? 2 : Shape<T, D>::kCtas)
    attn_decode_kernel(const __grid_constant__ DecodeParams dp, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v) {
  using S = Shape<T, D>;
  constexpr bool kF32 = S::kF32;
  constexpr int kKeys = S::kKeys, kWarpKeys = kKeys / kConsumers, NT = kWarpKeys / 8, KK = D / 16;
  constexpr int kHalves = kStack ? 1 : 2;  // rows g (and g + 8) of a quad
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[S::kStages], empty[S::kStages];
  __shared__ float top_s[kConsumers][16], sum_s[kConsumers][16];
  __shared__ int scan_s[kThreads / 32], place_s[2];
  __shared__ int redo_s[16];
  __shared__ uint64_t until_s;  // waits go on until then (wait_own)
  const AttnParams& p = dp.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const bool cut = dp.slots != nullptr;
  if (tid == 32 * kConsumers) {
    prefetch_map(&map_k);
    prefetch_map(&map_v);
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kConsumers);
    }
    fence_barrier_init();
  }
  pdl_wait();
  pdl_launch_dependents();
  if (tid == 0) move_on(&until_s);

  // ---- this CTA's run of the line: every thread adds up a block of sequences, then the one whose block
  // holds the run's beginning finds the sequence
  const int n_seqs = static_cast<int>(p.n_seqs), per = (n_seqs + kThreads - 1) / kThreads;
  const int s_lo = min(n_seqs, tid * per), s_hi = min(n_seqs, s_lo + per);
  int mine = 0;
  for (int s = s_lo; s < s_hi; ++s) mine += weight_of<T, D>(dp, s);
  int inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xFFFFFFFFu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) scan_s[warp] = inc;
  __syncthreads();
  int line = 0, before = inc - mine;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += scan_s[w];
    line += scan_s[w];
  }
  const int n_runs = min(static_cast<int>(gridDim.x), cut ? max(1, line / kMinRun) : line);
  if (static_cast<int>(blockIdx.x) >= n_runs || line == 0) {
    if (cut && tid == 0) dp.desc[blockIdx.x].parts = 0;
    return;
  }
  const Runs runs(line, n_runs);
  const int begin = static_cast<int>(runs.begin(blockIdx.x)), end = static_cast<int>(runs.begin(blockIdx.x + 1));
  if (begin >= before && begin < before + mine) {
    int at = begin - before, s = s_lo;
    if (per > 1)
      for (int n; (n = weight_of<T, D>(dp, s)) <= at; ++s) at -= n;
    place_s[0] = s;
    place_s[1] = at;
  }
  __syncthreads();
  Walk<T, D> walk;
  walk.start(place_s[0], place_s[1], end - begin);

  const uint32_t raw = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* ring = smem_raw + (base - raw);
  constexpr int kSlabRows = 8 * kHalves;
  float* o_s = reinterpret_cast<float*>(ring + S::kStages * 2 * S::kTileBytes);  // [warp][kSlabRows][D]
  int it = 0;  // tiles of the run so far

  if (warp == kConsumers) {
    // ---- producer: a lane per box of a tile (page by page), K and V
    const int boxes = kKeys / dp.box_rows, b = lane % boxes, panel = lane / boxes;
    bool ok = true;
    while (ok && walk.next(dp)) {
      const Rows& w = walk.w;
      auto row_of = [&](int tile) -> int32_t {
        const int pos = tile * kKeys + b * dp.box_rows;
        if (tile >= walk.to) return 0;
        if (!p.kv_len) return static_cast<int32_t>(w.c.begin + pos);
        const int64_t row = pos < w.see_all ? key_row(p, w.c, pos) : -1;
        return static_cast<int32_t>(row >= 0 ? row : p.n_pages * p.page_size);  // outside: zeros
      };
      int32_t row = row_of(walk.from);
      for (int tile = walk.from; tile < walk.to; ++tile) {
        const int st = it % S::kStages;
        const int32_t next = row_of(tile + 1);
        if (lane == 0) move_on(&until_s);
        if (it >= S::kStages) ok = wait_own(&empty[st], ((it / S::kStages) - 1) & 1, p.err, &until_s);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&full[st], 2 * S::kTileBytes);
        __syncwarp();
        uint8_t* dst = ring + st * 2 * S::kTileBytes + b * dp.box_rows * 128;
        for (int h = panel; h < S::kPanels; h += 32 / boxes) {
          constexpr int kPerPanel = 128 / static_cast<int>(sizeof(T));
          tma_load_3d(dst + h * S::kPanelBytes, &map_k, kPerPanel * h, walk.kvh, row, &full[st]);
          tma_load_3d(dst + S::kTileBytes + h * S::kPanelBytes, &map_v, kPerPanel * h, walk.kvh, row, &full[st]);
        }
        ++it;
        row = next;
      }
    }
    if (!ok)  // the copies in flight land before the shared memory is given back
      for (int i = max(0, it - S::kStages); i < it; ++i) wait_own(&full[i % S::kStages], (i / S::kStages) & 1, p.err, &until_s);
    return;
  }

  const float scale2 = p.scale * 1.4426950408889634f;
  const int key0 = warp * kWarpKeys, perm = (g >> 1) + 4 * (g & 1);
  bool ok = true, owner = false, first_part = true;
  while (walk.next(dp)) {
    const Rows& w = walk.w;
    const int kvh = walk.kvh;
    constexpr int kAcc = kStack ? 2 : 4;
    float acc[D / 8][kAcc];
    float top[kHalves], sum[kHalves];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int i = 0; i < kAcc; ++i) acc[n][i] = 0.f;
#pragma unroll
    for (int i = 0; i < kHalves; ++i) top[i] = -INFINITY, sum[i] = 0.f;
    // ---- queries as A fragments
    const T* qrow[2];
    int sees[kHalves];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = kStack ? g : g + 8 * i;
      const int token = r / p.group;
      const bool live = r < w.rows;
      qrow[i] = live ? static_cast<const T*>(p.q) + static_cast<int64_t>(w.c.begin + token) * p.q_stride +
                           static_cast<int64_t>(kvh * p.group + r - token * p.group) * p.head_dim
                     : nullptr;
      if (i < kHalves) sees[i] = live ? seen_by(w.c, w.c.begin + token) : 0;
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

    for (int tile = walk.from; tile < walk.to; ++tile, ++it) {
      const int st = it % S::kStages;
      if (ok) ok = wait_own(&full[st], (it / S::kStages) & 1, p.err, &until_s);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) continue;  // a wait gave up (recorded): no more work, but every barrier below is met
      const uint32_t ks = base + static_cast<uint32_t>(st) * (2 * S::kTileBytes), vs = ks + S::kTileBytes;
      const int j0 = tile * kKeys + key0;
      if (j0 + kWarpKeys > w.see_all) {
        // values behind the last position become zeros: 0 times what may lie there need not be 0
        const int keep = max(0, w.see_all - j0);
        for (int e = lane; e < (kWarpKeys - keep) * S::kPanels * 8; e += 32) {
          const int r = key0 + keep + e / (S::kPanels * 8), h = (e / 8) % S::kPanels;
          *reinterpret_cast<uint4*>(ring + (vs - base) + h * S::kPanelBytes + r * 128 + (e % 8) * 16) =
              make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();  // before the copy that fills this stage again
        __syncwarp();
      }
      // F32: the small products apart, and the large ones of 32 dims at a time, added to the score by an FP32
      // addition: the matrix instructions cut off where those round, at every step of a chain.
      float s[NT][4], s2[kF32 ? NT : 1][4], far[kF32 ? NT : 1][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[n][i] = 0.f;
          if constexpr (kF32) s2[n][i] = far[n][i] = 0.f;
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
                mma_tf32(s2[n], ah, kl[2 * h], kl[2 * h + 1]);
                mma_tf32(s2[n], al, kh[2 * h], kh[2 * h + 1]);
                mma_tf32(s[n], ah, kh[2 * h], kh[2 * h + 1]);
              }
            }
            if (kk % 2 == 1 && kk + 1 < KK) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                far[n][e] += s[n][e];
                s[n][e] = 0.f;
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
          for (int e = 0; e < 2; ++e) s[n][e] = (far[n][e] + s[n][e]) + ((far[n][e + 2] + s[n][e + 2] + s2[n][e]) + s2[n][e + 2]);
      } else if constexpr (kF32) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = (far[n][e] + s[n][e]) + s2[n][e];
      }
      // ---- softmax (base 2)
      const bool edge = j0 + kWarpKeys > w.see_first;
      float back[kHalves];
#pragma unroll
      for (int i = 0; i < kHalves; ++i) {
        const int limit = sees[i] - j0;
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
        back[i] = ex2(top[i] - ref);
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
        sum[i] = sum[i] * back[i] + add;
        if (!kF32 && __any_sync(0xFFFFFFFFu, moved)) {
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
        // instructions cut off instead of rounding, which over a long row would shrink it.
        uint32_t ph[NT][4], pl[NT][4];  // A fragments: k = t is key t, k = t + 4 key t + 4 of the eight
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (kStack) {
            split_tf32(s[n][0], ph[n][0], ph[n][1]);
            split_tf32(s[n][1], ph[n][2], ph[n][3]);
          } else {
            split_tf32(s[n][0], ph[n][0], pl[n][0]);
            split_tf32(s[n][2], ph[n][1], pl[n][1]);
            split_tf32(s[n][1], ph[n][2], pl[n][2]);
            split_tf32(s[n][3], ph[n][3], pl[n][3]);
          }
        }
#pragma unroll
        for (int dc = 0; dc < D / 32; ++dc) {  // column g of group (dc, i) is dim 32 dc + 4 perm + i
          float big[4][4] = {}, small[4][4] = {};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int r = key0 + 8 * n + t;  // and r + 4
            const uint32_t panel = vs + dc * S::kPanelBytes;
            const float4 v0 = lds128(panel + r * 128 + ((perm ^ (r & 7)) << 4));
            const float4 v1 = lds128(panel + (r + 4) * 128 + ((perm ^ ((r + 4) & 7)) << 4));
            const float a0[4] = {v0.x, v0.y, v0.z, v0.w}, a1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t h0, l0, h1, l1;
              split_tf32(a0[i], h0, l0);
              split_tf32(a1[i], h1, l1);
              mma_tf32(small[i], ph[n], l0, l1);
              if constexpr (!kStack) mma_tf32(small[i], pl[n], h0, h1);
              mma_tf32(big[i], ph[n], h0, h1);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < kAcc; ++e) {
              float& o = acc[4 * dc + i][e];
              if constexpr (kStack)
                o = fmaf(o, back[0], big[i][e] + (big[i][e + 2] + (small[i][e] + small[i][e + 2])));
              else
                o = fmaf(o, back[e >> 1], big[i][e] + small[i][e]);
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
    // ---- the warps' rows meet
    consumer_barrier();  // the rows of the part before have been read
#pragma unroll
    for (int i = 0; i < kHalves; ++i) {
      float v = sum[i];
      v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
      v += __shfl_xor_sync(0xFFFFFFFFu, v, 2);
      if (t == 0) {
        top_s[warp][g + 8 * i] = top[i];
        sum_s[warp][g + 8 * i] = v;
      }
      float* o = o_s + (warp * kSlabRows + g + 8 * i) * D;
      const auto value = [&](int n, int e) { return acc[n][2 * i + e]; };
      if constexpr (kF32) {  // dims 32 dc + 4 t + 16 e ..  + 3
#pragma unroll
        for (int n = 0; n < D / 8; n += 4)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<float4*>(o + slab_at<kF32>(g, 8 * n + 4 * t + 16 * e)) =
                make_float4(value(n, e), value(n + 1, e), value(n + 2, e), value(n + 3, e));
      } else {  // dims 8 n + 2 t, + 1
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<float2*>(o + slab_at<kF32>(g, 8 * n + 2 * t)) = make_float2(value(n, 0), value(n, 1));
      }
    }
    const bool whole = walk.from == 0 && walk.to == walk.all, uneven = whole && w.see_first < w.see_all;
    if (uneven && tid < 16) redo_s[tid] = 0;
    consumer_barrier();
    float* slot = whole ? nullptr : dp.slots + (static_cast<int64_t>(blockIdx.x) * 2 + (first_part ? 0 : 1)) * (16 * (D + 2));
    for (int e = tid; e < w.rows * D; e += 32 * kConsumers) {
      const int r = e / D, d = e % D;
      float mx = top_s[0][r];
#pragma unroll
      for (int x = 1; x < kConsumers; ++x) mx = fmaxf(mx, top_s[x][r]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      float v = 0.f, l = 0.f;
#pragma unroll
      for (int x = 0; x < kConsumers; ++x) {
        const float f = ex2(top_s[x][r] - ref);
        v += f * o_s[(x * kSlabRows + r) * D + slab_at<kF32>(r, d)];
        l += f * sum_s[x][r];
      }
      if (!whole) {
        slot[32 + e] = v;
        if (d == 0) {
          slot[r] = mx;
          slot[16 + r] = l;
        }
      } else if (d < p.head_dim) {
        if (store_row<T>(p, w, kvh, r, d, v, l) && uneven) redo_s[r] = 1;
      }
    }
    if (uneven) {
      consumer_barrier();
      if (warp == 0) redo_rows<T>(p, w, kvh, redo_s, &until_s);
    }
    if (warp == 0) {
      if (!whole && walk.from == 0) {  // a key head that is cut begins here: its last piece is in another run
        const int cta = static_cast<int>(runs.at(end - 1 + (walk.all - walk.to)));
        owner = true;
        if (lane == 0)
          dp.desc[blockIdx.x] = JoinDesc{walk.seq, kvh, first_part ? 0 : 1, cta - static_cast<int>(blockIdx.x) + 1,
                                         w.c.begin, w.c.end, w.c.kv_len, 0};
      }
    }
    first_part = false;
  }
  if (cut && tid == 0 && !owner) dp.desc[blockIdx.x].parts = 0;
}

// Joins the pieces of the key head whose first piece is at the end of CTA blockIdx.x's run:
// out = sum_x 2^(top_x - top) o_x / sum_x 2^(top_x - top) l_x. Rows blockIdx.y, blockIdx.y + gridDim.y, ..
// A group of threads takes every kGroups-th piece; its first kAhead pieces are loaded before the weights
// are known, so that few pieces cost one round of loads.
template <typename T, int D>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ DecodeParams dp) {
  constexpr int kGroups = 128 / (D / 4), kAhead = 2;  // a group reads one piece's row, 16 bytes a thread
  __shared__ float weight[kMaxCtas], part[kGroups][D], red[8];
  __shared__ int redo_s[16];
  const AttnParams& p = dp.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = tid / (D / 4), d = tid % (D / 4) * 4;
  if (tid < 16) redo_s[tid] = 0;
  pdl_wait();
  const JoinDesc j = dp.desc[blockIdx.x];
  if (j.parts <= 1) return;
  Rows w;
  w.c = Chunk{j.seq, j.begin, j.end, j.kv_len};
  w.rows = (j.end - j.begin) * p.group;
  w.see_first = seen_by(w.c, j.begin);
  w.see_all = seen_by(w.c, j.end - 1);
  constexpr int64_t kSlot = 16 * (D + 2);
  const float* slots = dp.slots + static_cast<int64_t>(blockIdx.x) * 2 * kSlot;
  auto slot = [&](int x) { return slots + (2 * x + (x == 0 ? j.first : 0)) * kSlot; };
  for (int r = blockIdx.y; r < w.rows; r += gridDim.y) {
    float4 ahead[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int x = group + k * kGroups;
      ahead[k] = x < j.parts ? *reinterpret_cast<const float4*>(slot(x) + 32 + r * D + d) : make_float4(0, 0, 0, 0);
    }
    float mx = -INFINITY, l = 0.f;
    for (int x = tid; x < j.parts; x += 128) mx = fmaxf(mx, weight[x] = slot(x)[r]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
    if (lane == 0) red[warp] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float ref = mx == -INFINITY ? 0.f : mx;
    for (int x = tid; x < j.parts; x += 128) {
      const float f = ex2(weight[x] - ref);
      weight[x] = f;
      l += f * slot(x)[16 + r];
    }
    l = warp_sum(l);
    if (lane == 0) red[4 + warp] = l;
    __syncthreads();
    l = (red[4] + red[5]) + (red[6] + red[7]);
    float4 acc = make_float4(0, 0, 0, 0);
    const auto add = [&](int x, const float4& v) {
      const float f = weight[x];
      acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (group + k * kGroups < j.parts) add(group + k * kGroups, ahead[k]);
#pragma unroll 4
    for (int x = group + kAhead * kGroups; x < j.parts; x += kGroups)
      add(x, *reinterpret_cast<const float4*>(slot(x) + 32 + r * D + d));
    *reinterpret_cast<float4*>(&part[group][d]) = acc;
    __syncthreads();
    if (tid < D && tid < p.head_dim) {
      float v = 0.f;
#pragma unroll
      for (int x = 0; x < kGroups; ++x) v += part[x][tid];
      if (store_row<T>(p, w, j.kvh, r, tid, v, l)) redo_s[r] = 1;
    }
    __syncthreads();
    if (redo_s[r] && w.see_first < w.see_all) {  // the same for every thread
      if (warp == 0) redo_rows<T>(p, w, j.kvh, redo_s);
      __syncthreads();
      if (tid == 0) redo_s[r] = 0;
    }
  }
}

template <typename T, int D, bool kStack>
int launch(const DecodeParams& dp, const CUtensorMap& mk, const CUtensorMap& mv, int ctas, cudaStream_t s) {
  using S = Shape<T, D>;
  const auto fn = attn_decode_kernel<T, D, kStack>;
  if (int st = ensure_smem_attr(reinterpret_cast<const void*>(fn), S::smem(kStack ? 8 : 16))) return st;
  const AttnParams& p = dp.a;
  cudaLaunchConfig_t cf{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cf.attrs = attr;
  cf.numAttrs = 1;
  cf.stream = s;
  cf.gridDim = dim3(static_cast<unsigned>(ctas));
  cf.blockDim = dim3(kThreads);
  cf.dynamicSmemBytes = S::smem(kStack ? 8 : 16);
  EFG_TRY_CUDA(cudaLaunchKernelEx(&cf, fn, dp, mk, mv), "attention launch");
  if (!dp.slots) return EFG_OK;
  const int64_t rows = std::min<int64_t>(kDecodeRows, std::min(p.kv_len ? p.max_new : p.n_rows, p.n_rows) * p.group);
  cf.gridDim = dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(std::min<int64_t>(rows, 8)));
  cf.blockDim = dim3(128);
  cf.dynamicSmemBytes = 0;
  EFG_TRY_CUDA(cudaLaunchKernelEx(&cf, attn_join_kernel<T, D>, dp), "attention launch");
  return EFG_OK;
}

int64_t max_keys_of(const AttnParams& p) { return p.kv_len ? p.max_pages * p.page_size : p.n_rows; }

// Whether key heads may be cut: not when each is at most a few tiles.
bool cuts(const AttnParams& p) { return max_keys_of(p) > kMinRun * 64; }

int ctas_of(const AttnParams& p, int sms) { return std::min(kMaxCtas, (p.head_dim <= 64 ? 3 : 2) * sms); }

template <typename T, int D>
int dispatch(int type, const AttnParams& p, int sms, void* work, cudaStream_t s) {
  using S = Shape<T, D>;
  static_assert(S::kCtas == (D == 64 ? 3 : 2));
  const int ctas = ctas_of(p, sms);
  DecodeParams dp;
  dp.a = p;
  dp.desc = static_cast<JoinDesc*>(work);
  dp.slots = cuts(p) ? reinterpret_cast<float*>(dp.desc + ctas) : nullptr;
  dp.box_rows = p.kv_len ? static_cast<int>(std::min<int64_t>(p.page_size, S::kKeys)) : S::kKeys;
  const int64_t kv_rows = p.kv_len ? p.n_pages * p.page_size : p.n_rows;
  CUtensorMap mk, mv;
  if (!encode_heads_map(&mk, type, p.k, p.head_dim, p.kv_heads, kv_rows, p.k_stride, 1, dp.box_rows) ||
      !encode_heads_map(&mv, type, p.v, p.head_dim, p.kv_heads, kv_rows, p.v_stride, 1, dp.box_rows))
    return fail(EFG_ECUDA, "attention: the driver rejects a tensor map");
  if constexpr (S::kF32) {
    if (std::min(p.kv_len ? p.max_new : p.n_rows, p.n_rows) * p.group <= 8) return launch<T, D, true>(dp, mk, mv, ctas, s);
  }
  return launch<T, D, false>(dp, mk, mv, ctas, s);
}

}  // namespace

bool attn_decode_takes(int type, const AttnParams& p) {
  if (p.k_stride == 0 || p.v_stride == 0) return false;
  if (p.kv_len && (p.n_pages == 0 || p.page_size < 8 || (p.page_size & (p.page_size - 1)))) return false;
  const int64_t max_new = std::min(p.kv_len ? p.max_new : p.n_rows, p.n_rows);
  // the line's weight is a 32-bit number
  if (p.n_seqs * p.kv_heads > 0x7FFFFFFFll / (max_keys_of(p) / 32 + 1 + kHeadCost)) return false;
  return attn_mma_takes(type, p) && max_new * p.group <= kDecodeRows;
}

size_t attn_decode_workspace(int, const AttnParams& p, int sms) {
  if (!cuts(p)) return 0;
  return static_cast<size_t>(ctas_of(p, sms)) * (sizeof(JoinDesc) + 2 * 16 * ((p.head_dim <= 64 ? 64 : 128) + 2) * sizeof(float));
}

int launch_attn_decode(int type, const AttnParams& p, int sms, void* work, cudaStream_t s) {
  const bool small = p.head_dim <= 64;
  if (type == EFG_F32) return small ? dispatch<float, 64>(type, p, sms, work, s) : dispatch<float, 128>(type, p, sms, work, s);
  if (type == EFG_F16) return small ? dispatch<__half, 64>(type, p, sms, work, s) : dispatch<__half, 128>(type, p, sms, work, s);
  return small ? dispatch<__nv_bfloat16, 64>(type, p, sms, work, s) : dispatch<__nv_bfloat16, 128>(type, p, sms, work, s);
}

}  // namespace efg
