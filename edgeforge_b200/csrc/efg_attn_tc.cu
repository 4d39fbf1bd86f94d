// efg_attn_tc.cu - attention of large row tiles (prompts, chunks) in 16-bit types on the 5th-generation
// tensor cores.
//
// One CTA per SM owns two 128-row tiles of one key head, each of floor(128 / group) tokens times the
// group's query heads (row = token * group + head), so a group shares its keys and the two tiles share
// every key and value tile (128 positions) that TMA brings into a ring. Per tile of keys and row tile:
//   S = Q K^T       tcgen05.mma, Q and K from shared memory, S (FP32) in TMEM;
//   P = 2^(S - ref) one softmax thread per row: TMEM -> 128 registers -> exponentials -> 16-bit P back
//                   into S's own TMEM columns;
//   O += P V        tcgen05.mma with A = P from TMEM, O (FP32) in TMEM.
// The two row tiles alternate: while one is in its softmax, the tensor cores work for the other.
// The reference value ref follows the running maximum lazily: it moves (and O is multiplied) only when
// the maximum has grown by more than 2^8, so weights stay below 256 and O is touched rarely.
//
// What bounds it: at head size 128 the two products of a 128 x 128 tile take 1024 tensor-core cycles and
// its 16384 exponentials 1024 cycles of the special function units; at 64 the exponentials are the
// bound. Part of them is therefore computed as polynomials on the FMA pipes (kPolyEvery below).
//
// Roles (12 warps): 0-3 and 4-7 softmax and epilogue of row tiles 0 and 1, 8 TMA, 9 MMA (10 and 11 only
// complete the warpgroup that gives its registers to the softmax: 2 x 128 x 208 + 128 x 80 of the
// launch's 384 x 168). TMEM (512 columns): S0 | S1 | O0 | O1. With few row tiles a cluster of CTAs splits the keys and joins the
// partial rows through distributed shared memory, in rank order.
#include <algorithm>

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "efg_attn.cuh"
#include "efg_attn_launch.h"
#include "efg_host.h"
#include "efg_tcgen05.cuh"

namespace cg = cooperative_groups;

namespace efg {
namespace {

constexpr int kThreads = 384, kTileKeys = 128, kTileRows = 128;
constexpr uint32_t kPanel = 128 * 128;  // 128 rows of 64 16-bit values, 128-byte swizzled
constexpr float kLazy = 8.f;            // powers of two that the maximum may grow before O is rescaled

template <int D>
constexpr int kv_stages() {
  return D == 64 ? 8 : 5;
}
template <int D>
constexpr size_t smem_bytes() {
  return 1024 + static_cast<size_t>(2 + kv_stages<D>()) * (D / 64) * kPanel;
}

// A value tile as the B operand of O += P V: keys run along K, so the tile (rows of keys, 64 dims of 128
// bytes, 128-byte swizzle) is MN-major: 64-dim panels kPanel apart, groups of 8 keys 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_values(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(kPanel >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Instruction descriptor: FP32 accumulator, A and B F16 or BF16, A K-major, B K-major or MN-major.
template <typename T>
constexpr uint32_t idesc_of(uint32_t N, bool b_mn) {
  const uint32_t fmt = std::is_same_v<T, __nv_bfloat16> ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn ? 1u : 0u) << 16) | ((N >> 3) << 17) | ((kTileRows >> 4) << 24);
}

// ---- MMA forms for a warp-uniform issue loop: executed by the thread whose `one` is set
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
}
template <bool kAdd>
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %0, 0;\n\t"
      "setp.ne.u32 p, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], %2, %3, %4, p;\n\t}" ::"r"(one),
      "r"(d), "l"(a), "l"(b), "r"(idesc), "n"(kAdd ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %0, 0;\n\t"
      "setp.ne.u32 p, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], %3, %4, p;\n\t}" ::"r"(one),
      "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t one, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.u32 q, %0, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}" ::"r"(one),
      "r"(smem_addr(bar))
      : "memory");
}

// ---- packed FP32 pairs
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x of two values on the FMA pipes: x = n + r with r in [-1/2, 1/2] (adding and subtracting 1.5 * 2^23
// rounds to an integer), 2^r as the degree-4 polynomial of least relative error on that interval
// (fitted for this kernel, error 2.6e-6, below the 16-bit rounding of the weight), n added to the
// exponent. x is held at -126 and above: smaller weights come out as 2^-126 instead.
__device__ __forceinline__ void poly_ex2(uint64_t x, float& a, float& b) {
  float xa, xb;
  unpair(x, xa, xb);
  x = pair(fmaxf(xa, -126.f), fmaxf(xb, -126.f));
  const uint64_t magic = pair(12582912.f, 12582912.f), t = add2(x, magic);
  const uint64_t n = add2(t, pair(-12582912.f, -12582912.f));
  const uint64_t r = fma2(n, pair(-1.f, -1.f), x);
  uint64_t y = fma2(pair(0.009570102207362652f, 0.009570102207362652f), r, pair(0.05591785907745361f, 0.05591785907745361f));
  y = fma2(y, r, pair(0.240247443318367f, 0.240247443318367f));
  y = fma2(y, r, pair(0.6931217908859253f, 0.6931217908859253f));
  y = fma2(y, r, pair(0.9999992847442627f, 0.9999992847442627f));
  float ya, yb, ta, tb;
  unpair(y, ya, yb);
  unpair(t, ta, tb);
  a = __uint_as_float(__float_as_uint(ya) + (__float_as_uint(ta) << 23));
  b = __uint_as_float(__float_as_uint(yb) + (__float_as_uint(tb) << 23));
}

// Ties the registers of a TMEM load to the point after its wait.
__device__ __forceinline__ void after_wait(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]),
                 "+r"(r[i + 6]), "+r"(r[i + 7]));
}

// One pair in kPolyEvery goes to the FMA pipes.
template <int D>
constexpr int kPolyEvery = D == 64 ? 2 : 4;

// Weights of 32 columns, packed to 16 bits; `total` collects the unrounded weights.
template <typename T, int D, bool kEdge>
__device__ __forceinline__ void weights32(const uint32_t* s, uint64_t scale, uint64_t nref, uint64_t& total,
                                          uint32_t (&out)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint64_t x = fma2(pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale, nref);
    float a, b;
    if (!kEdge && i % kPolyEvery<D> == kPolyEvery<D> - 1) {
      poly_ex2(x, a, b);
    } else {  // masked places (-inf) come out as exact zeros here
      unpair(x, a, b);
      a = ex2(a);
      b = ex2(b);
    }
    total = add2(total, pair(a, b));
    out[i] = pack2<T>(a, b);
  }
}

// All threads of the CTA, from inside their roles.
__device__ __forceinline__ void cta_barrier() {
  __syncwarp();
  asm volatile("bar.sync 0, %0;" ::"n"(kThreads) : "memory");
}

struct TcParams {
  AttnParams a;
  int tokens;         // tokens of a row tile
  int tiles_per_seq;  // pairs of row tiles per sequence at fixed places, or 0: found by a scan
  int box_rows;       // rows of one key / value box
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_kernel(const __grid_constant__ TcParams tp, const __grid_constant__ CUtensorMap map_q,
                   const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  constexpr int kPanels = D / 64, kStages = kv_stages<D>();
  constexpr uint32_t kTileBytes = kPanels * kPanel;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t q_full, kv_full[kStages], kv_empty[kStages], s_full[2], p_ready[2], o_full[2], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ int64_t scan_s[kThreads / 32 + 2];
  const AttnParams& p = tp.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cg::cluster_group cluster = cg::this_cluster();
  const int splits = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int kvh = blockIdx.y;
  const int64_t tile_id = blockIdx.x / splits;

  if (tp.tiles_per_seq == 0 && blockIdx.x == 0 && kvh == 0) check_offsets(p);
  RowTile rt;
  if (tp.tiles_per_seq > 0) {
    rt.seq = tile_id / tp.tiles_per_seq;
    rt.index = tp.tiles_per_seq - 1 - (tile_id - rt.seq * tp.tiles_per_seq);
  } else if (!find_tile<kThreads>(p, tile_id, 1, 2 * tp.tokens, scan_s, rt)) {
    return;  // uniform over the cluster, as the returns below
  }
  Chunk c;
  if (!chunk_of_seq(p, rt.seq, c)) return;
  const int m = c.end - c.begin;
  if (rt.index * 2 * tp.tokens >= m) return;
  const int token0 = static_cast<int>(rt.index) * 2 * tp.tokens;
  // tokens of the two row tiles, the keys that their last token sees, and tiles of keys of this CTA
  int tok[2], n[2];
  int see_last[2], see_all = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    tok[i] = max(0, min(tp.tokens, m - token0 - i * tp.tokens));
    see_last[i] = tok[i] ? seen_by(c, c.begin + token0 + i * tp.tokens + tok[i] - 1) : 0;
    see_all = max(see_all, see_last[i]);
  }
  const int tiles = (see_all + kTileKeys - 1) / kTileKeys;
  const int tile_begin = static_cast<int>(static_cast<int64_t>(tiles) * rank / splits);
  const int tile_end = static_cast<int>(static_cast<int64_t>(tiles) * (rank + 1) / splits);
  const int count = tile_end - tile_begin;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    n[i] = max(0, min(tile_end, (see_last[i] + kTileKeys - 1) / kTileKeys) - tile_begin);

  const uint32_t raw = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* q_s = smem_raw + (base - raw);
  uint8_t* ring = q_s + 2 * kTileBytes;
  if (tid == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&drained, 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 128);
      mbar_init(&o_full[i], 1);
    }
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 8 && count > 0) {
      // -------------------------------------------------------------- TMA
      if (lane == 0) {
        const int live = n[1] > 0 ? 2 : 1;
        mbar_arrive_expect_tx(&q_full, static_cast<uint32_t>(live * kPanels * tp.tokens * p.group) * 128u);
        for (int i = 0; i < live; ++i)
          for (int h = 0; h < kPanels; ++h)
            tma_load_3d(q_s + (i * kPanels + h) * kPanel, &map_q, 64 * h, kvh * p.group,
                        c.begin + token0 + i * tp.tokens, &q_full);
      }
      const int boxes = kTileKeys / tp.box_rows, b = lane % boxes, panel = lane / boxes;
      const bool mine = lane < boxes * kPanels;
      // first row of this lane's box in the tensor; outside of it (zero fill) behind the last position
      auto row_of = [&](int tile) -> int32_t {
        const int pos = tile * kTileKeys + b * tp.box_rows;
        if (!mine || tile >= tile_end) return 0;
        if (!p.kv_len) return c.begin + pos;
        const int64_t none = p.n_pages * p.page_size;
        const int64_t row = pos < see_all ? key_row(p, c, pos) : -1;
        return static_cast<int32_t>(row >= 0 ? row : none);
      };
      int32_t row = row_of(tile_begin);
      bool ok = true;
      int issued = 0;
      for (int j = 0; j < count && ok; ++j) {
        const int32_t next = row_of(tile_begin + j + 1);
        for (int kv = 0; kv < 2 && ok; ++kv) {
          const int item = 2 * j + kv, st = item % kStages;
          if (item >= kStages) ok = wait_own(&kv_empty[st], ((item / kStages) - 1) & 1, p.err);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&kv_full[st], kTileBytes);
          __syncwarp();
          if (mine)
            tma_load_3d(ring + st * kTileBytes + panel * kPanel + b * tp.box_rows * 128, kv ? &map_v : &map_k, 64 * panel,
                        kvh, row, &kv_full[st]);
          ++issued;
        }
        row = next;
      }
      // the copies in flight land before the shared memory is given back (all have, unless a wait gave up)
      if (!ok) {
        wait_own(&q_full, 0, p.err);
        for (int item = max(0, issued - kStages); item < issued; ++item)
          wait_own(&kv_full[item % kStages], (item / kStages) & 1, p.err);
      }
    } else if (warp == 9 && count > 0) {
      // -------------------------------------------------------------- MMA
      // The whole warp walks this code, so that addresses and descriptors stay warp-uniform (in uniform
      // registers); one elected thread issues. All 512 columns are this CTA's: TMEM addresses start at 0.
      constexpr uint32_t id_s = idesc_of<T>(kTileKeys, false), id_o = idesc_of<T>(D, true);
      const uint32_t one = elect_one();
      const uint32_t q_addr = base, ring_addr = base + 2 * kTileBytes;
      auto scores = [&](int i, int item) {
        const uint64_t dq = smem_desc_sw128(q_addr + i * kTileBytes);
        const uint64_t dk = smem_desc_sw128(ring_addr + (item % kStages) * kTileBytes);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint64_t adv = (ks / 4) * (kPanel >> 4) + (ks % 4) * 2;
          if (ks == 0)
            mma_ss<false>(one, 128 * i, dq + adv, dk + adv, id_s);
          else
            mma_ss<true>(one, 128 * i, dq + adv, dk + adv, id_s);
        }
        commit_if(one, &s_full[i]);
      };
      auto values = [&](int i, int item, uint32_t add) {
        const uint64_t dv = desc_values(ring_addr + (item % kStages) * kTileBytes);
        mma_ts(one, 256 + D * i, 128 * i, dv, id_o, add);
#pragma unroll
        for (int ks = 1; ks < kTileKeys / 16; ++ks)
          mma_ts(one, 256 + D * i, 128 * i + 8 * ks, dv + ks * (2048 >> 4), id_o, 1u);
      };
      bool ok = wait_own(&q_full, 0, p.err) && wait_own(&kv_full[0], 0, p.err);
      if (ok) {
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (n[i] > 0) scores(i, 0);
        commit_if(one, &kv_empty[0]);
      }
      for (int j = 0; j < count && ok; ++j) {
        const int vi = 2 * j + 1, ki = 2 * j + 2;
        ok = wait_own(&kv_full[vi % kStages], (vi / kStages) & 1, p.err);
        if (ok && j + 1 < count) ok = wait_own(&kv_full[ki % kStages], (ki / kStages) & 1, p.err);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!ok || j >= n[i]) continue;
          ok = wait_own(&p_ready[i], j & 1, p.err);
          if (!ok) continue;
          tc_fence_after();
          values(i, vi, j > 0);
          if (j + 1 < n[i])
            scores(i, ki);
          else
            commit_if(one, &o_full[i]);
        }
        if (!ok) break;
        commit_if(one, &kv_empty[vi % kStages]);
        if (j + 1 < count) commit_if(one, &kv_empty[ki % kStages]);
      }
      commit_if(one, &drained);  // no MMA runs on when the TMEM is given back, also after a wait gave up
      __syncwarp();
      mbar_drain(&drained, 0, p.err);
    }
    if (splits > 1) {  // the joining of the softmax warps below
      cta_barrier();
      cluster.sync();
      cluster.sync();
    }
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int i = warp >> 2, r = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t s_addr = tmem + lanes + 128 * i, o_addr = tmem + lanes + 256 + D * i;
    const int token = r / p.group;  // of the row tile
    const bool live = token < tok[i];
    const int sees = live ? seen_by(c, c.begin + token0 + i * tp.tokens + token) : 0;
    const int see_first = tok[i] ? seen_by(c, c.begin + token0 + i * tp.tokens) : 0;
    const float scale2 = p.scale * 1.4426950408889634f;
    const uint64_t scale_pair = pair(scale2, scale2);
    uint64_t total = pair(0.f, 0.f);
    float ref = 0.f;
    bool ok = true;
    for (int j = 0; j < n[i]; ++j) {
      ok = wait_own(&s_full[i], j & 1, p.err);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      tc_fence_after();
      uint32_t s[128];
#pragma unroll
      for (int q = 0; q < 4; ++q) tmem_ld32(s_addr + 32 * q, s + 32 * q);
      tmem_wait_ld();
#pragma unroll
      for (int q = 0; q < 4; ++q) after_wait(s + 32 * q);
      const int key0 = (tile_begin + j) * kTileKeys;
      const bool edge = key0 + kTileKeys > see_first;
      if (edge) {
        const int limit = sees - key0;
#pragma unroll
        for (int k = 0; k < 128; ++k)
          if (k >= limit) s[k] = 0xFF800000u;  // -inf
      }
      float mx[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) mx[q] = fmaxf(__uint_as_float(s[q]), __uint_as_float(s[q + 4]));
#pragma unroll
      for (int k = 8; k < 128; k += 8)
#pragma unroll
        for (int q = 0; q < 4; ++q) mx[q] = max3(mx[q], __uint_as_float(s[k + q]), __uint_as_float(s[k + q + 4]));
      const float high = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
      if (j == 0) {
        ref = high == -INFINITY ? 0.f : high;
      } else {
        const bool move = high - ref > kLazy;
        if (__any_sync(0xFFFFFFFFu, move)) {  // the MMAs of the tile before are done: S of this one follows them
          const float back = move ? ex2(ref - high) : 1.f;
          if (move) ref = high;
          float ta, tb;
          unpair(total, ta, tb);
          total = pair(ta * back, tb * back);
#pragma unroll 1
          for (int q = 0; q < D / 32; ++q) {
            uint32_t o[32];
            tmem_ld32(o_addr + 32 * q, o);
            tmem_wait_ld();
            after_wait(o);
            uint32_t lo[16], hi[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              lo[e] = __float_as_uint(__uint_as_float(o[e]) * back);
              hi[e] = __float_as_uint(__uint_as_float(o[e + 16]) * back);
            }
            tmem_st16(o_addr + 32 * q, lo);
            tmem_st16(o_addr + 32 * q + 16, hi);
          }
        }
      }
      const uint64_t nref = pair(-ref, -ref);
      if (edge) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t w[16];
          weights32<T, D, true>(s + 32 * q, scale_pair, nref, total, w);
          tmem_st16(s_addr + 16 * q, w);
        }
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t w[16];
          weights32<T, D, false>(s + 32 * q, scale_pair, nref, total, w);
          tmem_st16(s_addr + 16 * q, w);
        }
      }
      if (key0 + kTileKeys > see_all) {
        // values behind the last position: whatever lies there would meet weights of zero, and 0 times
        // infinity is NaN, so it becomes zero
        const int item = 2 * j + 1, st = item % kStages;
        ok = wait_own(&kv_full[st], (item / kStages) & 1, p.err);
        if (ok && key0 + r >= see_all) {
#pragma unroll
          for (int h = 0; h < kPanels; ++h) {
            uint4* row = reinterpret_cast<uint4*>(ring + st * kTileBytes + h * kPanel + r * 128);
#pragma unroll
            for (int e = 0; e < 8; ++e) row[e] = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async();
        if (!__all_sync(0xFFFFFFFFu, ok)) break;
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_ready[i]);
    }
    float ta, tb;
    unpair(total, ta, tb);
    const float row_sum = ta + tb;
    if (ok && n[i] > 0) ok = wait_own(&o_full[i], 0, p.err);
    tc_fence_after();
    ok = __all_sync(0xFFFFFFFFu, ok);

    if (splits == 1) {
      const float inv = sees > 0 && row_sum != 0.f ? 1.f / row_sum : 0.f;
      const int64_t row = c.begin + token0 + i * tp.tokens + token;
      const int head = kvh * p.group + r - token * p.group;
      T* out = static_cast<T*>(p.out) + (row * p.heads + head) * p.head_dim;
      bool finite = true;
#pragma unroll 1
      for (int q = 0; q < D / 32; ++q) {
        uint32_t o[32];
        if (n[i] > 0) {
          tmem_ld32(o_addr + 32 * q, o);
          tmem_wait_ld();
          after_wait(o);
        }
        if (live && ok) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float a = inv == 0.f ? 0.f : __uint_as_float(o[e + 2 * x]) * inv;
              const float b = inv == 0.f ? 0.f : __uint_as_float(o[e + 2 * x + 1]) * inv;
              finite = finite && fabsf(a) <= 3.402823466e38f && fabsf(b) <= 3.402823466e38f;
              w[x] = pack2<T>(a, b);
            }
            if (32 * q + e < p.head_dim)
              *reinterpret_cast<uint4*>(out + 32 * q + e) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      // a row may not be reached by what lies at positions it does not see
      uint32_t redo = __ballot_sync(0xFFFFFFFFu, live && ok && !finite && sees < see_all);
      if (redo) {
        // scratch for one query: this warp's part of the Q area, whose MMAs are done
        float* scratch = reinterpret_cast<float*>(q_s + i * kTileBytes) + (warp & 3) * 256;
        __syncwarp();
        while (redo) {
          const int l = __ffs(redo) - 1;
          redo &= redo - 1;
          const int64_t row_l = __shfl_sync(0xFFFFFFFFu, row, l);
          const int head_l = __shfl_sync(0xFFFFFFFFu, head, l);
          if (reached_from_behind<T>(p, c, row_l, kvh, see_all)) attend_row<T>(p, c, row_l, head_l, scratch);
        }
      }
    }
    if (splits > 1) {
      // partial rows to shared memory (every operand there has been used): row r of [256][D] FP32 with its
      // 16-byte chunks rotated by r, so that a warp's rows fall into different banks
      cta_barrier();
      float* o_s = reinterpret_cast<float*>(q_s);
      float *part_top = o_s + 256 * D, *part_sum = part_top + 256;
      int* redo_s = reinterpret_cast<int*>(part_sum + 256);
      redo_s[tid] = 0;
      // a row that saw none of these keys takes no part
      part_top[tid] = row_sum == 0.f ? -INFINITY : ref;
      part_sum[tid] = row_sum;
#pragma unroll 1
      for (int q = 0; q < D / 32; ++q) {
        uint32_t o[32];
        if (n[i] > 0) {
          tmem_ld32(o_addr + 32 * q, o);
          tmem_wait_ld();
          after_wait(o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<uint4*>(o_s + tid * D + ((8 * q + e + r) % (D / 4)) * 4) =
              make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
      }
      __syncwarp();
      cluster.sync();
      // this CTA's share of the rows, 8 dims a thread, partials in rank order
      const int share = 256 / splits, r_lo = rank * share;
      for (int e = tid; e < share * (D / 8); e += 256) {
        const int rr = r_lo + e / (D / 8), d = (e % (D / 8)) * 8, ti = rr >> 7, tr = rr & 127, tt = tr / p.group;
        if (tt >= tok[ti] || d >= p.head_dim) continue;
        float mx = -INFINITY;
        for (int w = 0; w < splits; ++w) mx = fmaxf(mx, cluster.map_shared_rank(part_top, w)[rr]);
        const float high = mx == -INFINITY ? 0.f : mx;
        float acc[8] = {}, l = 0.f;
        for (int w = 0; w < splits; ++w) {
          const float f = ex2(cluster.map_shared_rank(part_top, w)[rr] - high);
          l += f * cluster.map_shared_rank(part_sum, w)[rr];
          const float* o = cluster.map_shared_rank(o_s, w) + rr * D;
          const float4 a = *reinterpret_cast<const float4*>(o + ((d / 4 + tr) % (D / 4)) * 4);
          const float4 b = *reinterpret_cast<const float4*>(o + ((d / 4 + 1 + tr) % (D / 4)) * 4);
          acc[0] += f * a.x, acc[1] += f * a.y, acc[2] += f * a.z, acc[3] += f * a.w;
          acc[4] += f * b.x, acc[5] += f * b.y, acc[6] += f * b.z, acc[7] += f * b.w;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint32_t w[4];
        bool finite = true;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          acc[2 * x] *= inv;
          acc[2 * x + 1] *= inv;
          finite = finite && fabsf(acc[2 * x]) <= 3.402823466e38f && fabsf(acc[2 * x + 1]) <= 3.402823466e38f;
          w[x] = pack2<T>(acc[2 * x], acc[2 * x + 1]);
        }
        const int64_t row = c.begin + token0 + ti * tp.tokens + tt;
        const int head = kvh * p.group + tr - tt * p.group;
        *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (row * p.heads + head) * p.head_dim + d) =
            make_uint4(w[0], w[1], w[2], w[3]);
        if (!finite) redo_s[rr] = 1;
      }
      __syncwarp();
      cluster.sync();  // every peer has read this CTA's partials; redo_s is complete
      float* scratch = o_s + warp * 256;
      for (int x = warp; x < share; x += 8) {
        const int rr = r_lo + x, ti = rr >> 7, tr = rr & 127, tt = tr / p.group;
        if (tt >= tok[ti] || !redo_s[rr]) continue;
        const int64_t row = c.begin + token0 + ti * tp.tokens + tt;
        if (seen_by(c, static_cast<int>(row)) < see_all && reached_from_behind<T>(p, c, row, kvh, see_all))
          attend_row<T>(p, c, row, kvh * p.group + tr - tt * p.group, scratch);
      }
    }
  }
  tc_fence_before();
  cta_barrier();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

template <typename T, int D>
int launch(const AttnParams& p, int64_t max_new, int64_t max_keys, int sms, cudaStream_t s) {
  TcParams tp;
  tp.a = p;
  tp.tokens = kTileRows / p.group;
  const int type = std::is_same_v<T, __nv_bfloat16> ? EFG_BF16 : EFG_F16;
  const int64_t kv_rows = p.kv_len ? p.n_pages * p.page_size : p.n_rows;
  tp.box_rows = p.kv_len ? static_cast<int>(std::min<int64_t>(p.page_size, kTileKeys)) : kTileKeys;
  CUtensorMap mq, mk, mv;
  if (!encode_heads_map(&mq, type, p.q, p.head_dim, p.heads, p.n_rows, p.q_stride, p.group, tp.tokens) ||
      !encode_heads_map(&mk, type, p.k, p.head_dim, p.kv_heads, kv_rows, p.k_stride, 1, tp.box_rows) ||
      !encode_heads_map(&mv, type, p.v, p.head_dim, p.kv_heads, kv_rows, p.v_stride, 1, tp.box_rows))
    return fail(EFG_ECUDA, "attention: the driver rejects a tensor map");
  const int64_t pair_tokens = 2 * tp.tokens, per_seq = (max_new + pair_tokens - 1) / pair_tokens;
  const int64_t fixed = p.n_seqs * per_seq, bound = p.n_rows / pair_tokens + p.n_seqs;
  const int64_t tiles = std::min(fixed, bound);
  tp.tiles_per_seq = fixed <= bound ? static_cast<int>(per_seq) : 0;
  // Split the keys while the row tiles leave half of the SMs idle and every split keeps 4 key tiles.
  int splits = 1;
  while (splits < 8 && tiles * p.kv_heads * splits * 2 <= sms && max_keys >= 2 * splits * 4 * kTileKeys) splits *= 2;
  if (tiles * splits > 0x7FFFFFFFll) return fail(EFG_EINVAL, "attention: too many rows");
  const auto fn = attn_tc_kernel<T, D>;
  if (int st = ensure_smem_attr(reinterpret_cast<const void*>(fn), smem_bytes<D>())) return st;
  cudaLaunchConfig_t cf{};
  cf.gridDim = dim3(static_cast<unsigned>(tiles * splits), static_cast<unsigned>(p.kv_heads));
  cf.blockDim = dim3(kThreads);
  cf.dynamicSmemBytes = smem_bytes<D>();
  cf.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(splits), 1, 1};
  cf.attrs = attr;
  cf.numAttrs = 1;
  EFG_TRY_CUDA(cudaLaunchKernelEx(&cf, fn, tp, mq, mk, mv), "attention launch");
  return EFG_OK;
}

}  // namespace

bool attn_tc_takes(int type, const AttnParams& p) {
  if (type == EFG_F32 || !(p.scale > 0.f) || p.group > kTileRows || reinterpret_cast<uintptr_t>(p.out) % 16) return false;
  if (p.q_stride == 0 || p.k_stride == 0 || p.v_stride == 0) return false;
  if (p.kv_len) {  // whole boxes of a page, whole 8-row groups of the swizzle
    if (p.n_pages == 0 || p.page_size < 8 || (p.page_size & (p.page_size - 1))) return false;
  }
  const int64_t max_new = p.kv_len ? std::min(p.max_new, p.n_rows) : p.n_rows;
  return attn_mma_takes(type, p) && max_new * p.group > 64;
}

int launch_attn_tc(int type, const AttnParams& p, int sms, cudaStream_t s) {
  const int64_t max_new = p.kv_len ? std::min(p.max_new, p.n_rows) : p.n_rows;
  const int64_t max_keys = p.kv_len ? p.max_pages * p.page_size : p.n_rows;
  if (type == EFG_F16)
    return p.head_dim <= 64 ? launch<__half, 64>(p, max_new, max_keys, sms, s)
                            : launch<__half, 128>(p, max_new, max_keys, sms, s);
  return p.head_dim <= 64 ? launch<__nv_bfloat16, 64>(p, max_new, max_keys, sms, s)
                          : launch<__nv_bfloat16, 128>(p, max_new, max_keys, sms, s);
}

}  // namespace efg
