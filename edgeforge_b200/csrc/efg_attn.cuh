// efg_attn.cuh - what the attention kernels share: the call's parameters, typed loads and the
// row-by-row softmax that every other kernel falls back to.
#pragma once

#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "efg_device.cuh"
#include "efg_paged.cuh"

namespace efg {

struct AttnParams {
  void* out;                 // [n_rows][heads][head_dim]
  const void* q;             // rows of q_stride elements
  const void *k, *v;         // prompt: rows of k_stride / v_stride elements; paged: the pools
  const int32_t* cu;         // [n_seqs + 1] first row of each sequence
  const int32_t* kv_len;     // paged: positions of each sequence, the new ones included; null: prompt
  const int32_t* table;      // paged: [n_seqs][max_pages]
  int64_t q_stride, k_stride, v_stride;
  int64_t n_rows, n_seqs, n_pages, max_pages, page_size, max_new;
  int page_shift;            // page_size = 1 << page_shift, or -1
  int heads, kv_heads, group, head_dim;
  float scale;
  int *err, *checks;         // for waits that give up, for offsets, lengths and pages that make no sense
};

__device__ __forceinline__ float attn_widen(float v) { return v; }
__device__ __forceinline__ float attn_widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float attn_widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T attn_narrow(float v) {
  if constexpr (sizeof(T) == 4)
    return v;
  else if constexpr (std::is_same_v<T, __half>)
    return __float2half_rn(v);
  else
    return __float2bfloat16_rn(v);
}

// The chunk of the packed batch that a row belongs to.
struct Chunk {
  int32_t seq, begin, end;  // sequence and its rows [begin, end)
  int32_t kv_len;           // its positions
};

__device__ __forceinline__ int32_t seen_by(const Chunk& c, int32_t row) { return visible_keys(row, c.end, c.kv_len); }

// False for rows behind the last sequence and for offsets that make no sense (recorded).
__device__ __forceinline__ bool chunk_of_seq(const AttnParams& p, int64_t s, Chunk& c) {
  c.seq = static_cast<int32_t>(s);
  c.begin = p.cu[s];
  c.end = p.cu[s + 1];
  if (c.begin < 0 || c.end > p.n_rows || c.end < c.begin || (p.kv_len && c.end - c.begin > p.max_new)) {
    record_error(p.checks, EFG_EINVAL);
    return false;
  }
  c.kv_len = c.end - c.begin;
  if (p.kv_len) {
    c.kv_len = p.kv_len[s];
    if (c.kv_len < 0 || c.kv_len > p.max_pages * p.page_size) {
      record_error(p.checks, EFG_EINVAL);
      return false;
    }
  }
  return true;
}

// Looks at every offset once (one CTA's threads): kernels that find a row's sequence by search may miss a
// bad one.
__device__ __forceinline__ void check_offsets(const AttnParams& p) {
  for (int64_t s = threadIdx.x; s < p.n_seqs; s += blockDim.x)
    if (p.cu[s] < 0 || p.cu[s + 1] < p.cu[s] || p.cu[s + 1] > p.n_rows) record_error(p.checks, EFG_EINVAL);
}

// Offset of the key (stride k_stride) of position j of the chunk's sequence, in rows of kv_heads *
// head_dim elements for pages; -1 where the block table has no valid page (recorded).
__device__ __forceinline__ int64_t key_row(const AttnParams& p, const Chunk& c, int32_t j) {
  if (!p.kv_len) return static_cast<int64_t>(c.begin) + j;
  // a position fits 31 bits, so the division (where the page size is no power of two) is a 32-bit one
  const uint32_t pos = static_cast<uint32_t>(j), size = static_cast<uint32_t>(p.page_size);
  const uint32_t pi = p.page_shift >= 0 ? pos >> p.page_shift : pos / size;
  const int32_t page = p.table[static_cast<int64_t>(c.seq) * p.max_pages + pi];
  if (!page_ok(page, p.n_pages)) {
    record_error(p.checks, EFG_EINVAL);
    return -1;
  }
  return page * p.page_size + (pos - pi * size);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Waits of a CTA for its own copies, MMAs and threads: an error that another CTA recorded does not end
// them, only *until (shared memory), the time limit that the CTA's warps have in common: the warp that issues
// the copies moves it on with every tile, and so does a warp that computes rows of a long sequence alone.
// (A start time in each wait beside that took 3 % of ragged 16-bit prompts.)
__device__ __forceinline__ void move_on(uint64_t* until) {
  *reinterpret_cast<volatile uint64_t*>(until) = globaltimer_ns() + kWaitTimeoutNs;
}
__device__ __forceinline__ bool wait_own(uint64_t* bar, uint32_t parity, int* err, const uint64_t* until) {
  if (mbar_try_wait(bar, parity)) return true;
#pragma unroll 1
  for (uint32_t i = 0;; ++i) {
    if (mbar_try_wait_sleep(bar, parity, 2000u)) return true;
    if ((i & 15u) == 15u && globaltimer_ns() > *reinterpret_cast<const volatile uint64_t*>(until)) {
      record_error(err, EFG_ETIMEOUT);
      return false;
    }
  }
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}

// A line of `line` weights cut into n runs that differ by one at most.
struct Runs {
  uint32_t runs, size, longer;  // the first `longer` runs weigh size + 1
  __device__ __forceinline__ Runs(uint32_t line, uint32_t n) : runs(n), size(line / n), longer(line - line / n * n) {}
  __device__ __forceinline__ uint32_t begin(uint32_t i) const { return i * size + min(i, longer); }
  __device__ __forceinline__ uint32_t at(uint32_t place) const {  // the run that holds a place
    const uint32_t split = longer * (size + 1);
    return place < split ? place / (size + 1) : longer + (place - split) / size;
  }
};

// The tile of rows a CTA owns: its sequence and its place among the sequence's tiles.
struct RowTile {
  int64_t seq, index;
};

// Tile `want` when every sequence has ceil(rows * mul / div) tiles, in order; the tiles of one
// sequence come last to first (the last one of a prompt is the longest). The whole CTA (kThreads
// threads) calls it; `scan` is shared, kThreads / 32 + 2 entries. False behind the last tile.
template <int kThreads>
__device__ bool find_tile(const AttnParams& p, int64_t want, int64_t mul, int64_t div, int64_t* scan, RowTile& t) {
  constexpr int kWarps = kThreads / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t base = 0;
  for (int64_t s0 = 0; s0 < p.n_seqs; s0 += kThreads) {
    int64_t n = 0;
    if (s0 + tid < p.n_seqs) {
      const int64_t m = static_cast<int64_t>(p.cu[s0 + tid + 1]) - p.cu[s0 + tid];
      // lengths that make no sense get one tile, whose CTA records them
      n = m < 0 || m > p.n_rows ? 1 : (m * mul + div - 1) / div;
    }
    int64_t inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    int64_t before = base, total = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    if (want >= before + inc - n && want < before + inc) {
      scan[kWarps] = s0 + tid;
      scan[kWarps + 1] = before + inc - 1 - want;
    }
    __syncthreads();
    if (want < base + total) {
      t.seq = scan[kWarps];
      t.index = scan[kWarps + 1];
      return true;
    }
    base += total;
  }
  return false;
}

// One warp computes one row of one query head: 32 keys at a time, a lane per dim of keys and values, running maximum and
// sum of the softmax in FP32. Bound by the latency of its loads, so they are unconditional (of a place that is valid in
// any case) and kAhead keys' are in flight; more of them, or 8 lanes a key, would take registers that the kernels
// that call this have none left of (64 FP32 rows of a decode step: 44.9 -> 56.6 us). A key behind the row's last visible
// one is never read, so what lies there (stale, infinite or NaN) cannot reach the row. head_dim <= 32 N; lane l holds
// dims l, l + 32, .. of the query.
template <typename T, int N>
__device__ __forceinline__ void attend_row_of(const AttnParams& p, const Chunk& c, int64_t row, int head, uint64_t* until) {
  constexpr int kAhead = N == 8 ? 2 : 16 / N;
  const int lane = threadIdx.x & 31, D = p.head_dim, kvh = head / p.group;
  const int32_t count = seen_by(c, static_cast<int32_t>(row));
  const T* q = static_cast<const T*>(p.q) + row * p.q_stride + static_cast<int64_t>(head) * D;
  float qv[N], acc[N] = {}, top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) qv[i] = lane + 32 * i < D ? attn_widen(q[lane + 32 * i]) : 0.f;
  const float to_base2 = p.scale * 1.4426950408889634f;
  for (int32_t j0 = 0; j0 < count; j0 += 32) {
    if (until && lane == 0) move_on(until);
    int64_t kr = -1;  // of key j0 + lane
    if (j0 + lane < count) kr = key_row(p, c, j0 + lane);
    const uint32_t good = __ballot_sync(0xFFFFFFFFu, kr >= 0);
    if (good == 0) continue;
    const int64_t some = __shfl_sync(0xFFFFFFFFu, kr, __ffs(good) - 1);
    if (kr < 0) kr = some;
    const int n = min(32, count - j0);
    const auto load = [&](const void* base, int64_t stride, int t, T (&x)[kAhead][N]) {  // keys t .., this lane's dims
#pragma unroll
      for (int y = 0; y < kAhead; ++y) {
        const T* at = static_cast<const T*>(base) + __shfl_sync(0xFFFFFFFFu, kr, t + y) * stride + static_cast<int64_t>(kvh) * D;
#pragma unroll
        for (int i = 0; i < N; ++i) x[y][i] = at[min(lane + 32 * i, D - 1)];
      }
    };
    float dot = 0.f;
#pragma unroll 1
    for (int t = 0; t < n; t += kAhead) {
      T x[kAhead][N];
      load(p.k, p.k_stride, t, x);
#pragma unroll
      for (int y = 0; y < kAhead; ++y) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (lane + 32 * i < D) s = fmaf(qv[i], attn_widen(x[y][i]), s);
        s = warp_sum(s);
        if (lane == t + y) dot = s;
      }
    }
    const bool valid = good >> lane & 1;
    const float sc = valid ? dot * to_base2 : -INFINITY;
    float m = sc;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float t = __shfl_xor_sync(0xFFFFFFFFu, m, o);
      m = (t != t || m != m) ? NAN : fmaxf(m, t);  // a NaN score makes the row NaN
    }
    const float high = (m != m || top != top) ? NAN : fmaxf(top, m);
    // nothing visible so far (every score -inf): keep the sums at zero
    const float ref = high == -INFINITY ? 0.f : high;
    const float w = valid ? exp2f(sc - ref) : 0.f;
    const float back = exp2f(top - ref);
    sum = sum * back + warp_sum(w);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= back;
    top = high;
#pragma unroll 1
    for (int t = 0; t < n; t += kAhead) {
      T x[kAhead][N];
      load(p.v, p.v_stride, t, x);
#pragma unroll
      for (int y = 0; y < kAhead; ++y) {
        const float wt = __shfl_sync(0xFFFFFFFFu, w, t + y);
        if (good >> (t + y) & 1) {
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] = fmaf(wt, attn_widen(x[y][i]), acc[i]);
        }
      }
    }
  }
  T* out = static_cast<T*>(p.out) + (row * p.heads + head) * D;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing is zeros
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane + 32 * i < D) out[lane + 32 * i] = attn_narrow<T>(acc[i] * inv);
}
// The same for any head size; *until (null: none) is moved on for the waits of the CTA's other warps (wait_own).
template <typename T>
__device__ __noinline__ void attend_row(const AttnParams& p, const Chunk& c, int64_t row, int head, uint64_t* until = nullptr) {
  if (p.head_dim <= 64)
    attend_row_of<T, 2>(p, c, row, head, until);
  else if (p.head_dim <= 128)
    attend_row_of<T, 4>(p, c, row, head, until);
  else
    attend_row_of<T, 8>(p, c, row, head, until);
}

// Whether a non-finite value of the KV head lies at a position that the row does not see, but
// that was in a tile with positions it sees (up to `end`): 0 times it is NaN in a matrix product.
// One warp; every lane gets the answer.
template <typename T>
__device__ __noinline__ bool reached_from_behind(const AttnParams& p, const Chunk& c, int64_t row, int kvh, int32_t end) {
  const int lane = threadIdx.x & 31;
  bool bad = false;
  for (int32_t j = seen_by(c, static_cast<int32_t>(row)); j < end; ++j) {
    const int64_t vr = key_row(p, c, j);
    if (vr < 0) continue;
    const T* v = static_cast<const T*>(p.v) + vr * p.v_stride + static_cast<int64_t>(kvh) * p.head_dim;
    // (from 2^127 on the upper part of a split FP32 value may round to infinity)
    for (int d = lane; d < p.head_dim; d += 32) bad = bad || !(fabsf(attn_widen(v[d])) < 1.701411835e38f);
  }
  return __any_sync(0xFFFFFFFFu, bad);
}

}  // namespace efg
