// efg_paged.cu - one serving step's bookkeeping and cache writes:
//   page_plan   lengths + free list -> block tables, slot map, positions, prefix sums;
//   page_store  RoPE of the step's queries and keys, keys and values to their cache slots.
// The index arithmetic is in efg_paged.cuh.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/efg.h"
#include "efg_device.cuh"
#include "efg_host.h"
#include "efg_paged.cuh"

namespace efg {
namespace {

// ---------------------------------------------------------------- step planning
struct PlanParams {
  int32_t* table;
  int32_t *slots, *positions, *cu, *kv_len, *taken;
  const int32_t *cached, *fresh, *free;
  int64_t max_pages, n_rows, n_seqs, n_free, n_pages, page_size, most, rows_per_cta;  // most: positions of a sequence
  int* checks;
};

constexpr int kPlanThreads = 512;

struct Pair64 {
  int64_t rows, need;
};

__device__ __forceinline__ Pair64 operator+(Pair64 a, Pair64 b) { return Pair64{a.rows + b.rows, a.need + b.need}; }

// Exclusive prefix sums over the CTA's threads; `total` is the sum over all of them.
__device__ __forceinline__ Pair64 block_prefix(Pair64 v, Pair64* warp_sums, Pair64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Pair64 inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Pair64 up{__shfl_up_sync(0xFFFFFFFFu, inc.rows, o), __shfl_up_sync(0xFFFFFFFFu, inc.need, o)};
    if (lane >= o) inc = inc + up;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  Pair64 before{0, 0};
  total = Pair64{0, 0};
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w == warp) before = total;
    total = total + warp_sums[w];
  }
  return Pair64{before.rows + inc.rows - v.rows, before.need + inc.need - v.need};
}

// One launch, no hand-over between CTAs: every CTA walks the sequences in chunks of kChunk (kPerThread per
// thread; two prefix sums per chunk: packed rows and fresh pages) up to the end of its own range of
// rows, and fills that range: a row finds its sequence by bisection among the chunk's row offsets in
// shared memory. CTA 0 also writes the per-sequence outputs. The row that opens a page writes the block
// table's entry (fresh pages start at multiples of page_size). Bound by latency: the bytes (8 per row,
// 12 per sequence, 8 per page) are a few MB at most, and a second launch for the prefix sums would
// cost more than repeating them per CTA does. Measured: 4.2 us for 8 single tokens; 2048 sequences with
// 297763 new tokens 13.0 us with one sequence per thread and 64-bit divisions, 7.3 us as it is.
constexpr int kPerThread = 4, kChunk = kPlanThreads * kPerThread;

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PlanParams p) {
  __shared__ int32_t row0[kChunk];   // first packed row of each sequence of the chunk (n_rows where it passes that)
  __shared__ int32_t page0[kChunk];  // its first fresh page in the free list; -1: not served
  __shared__ int32_t have_s[kChunk], cached_s[kChunk];
  __shared__ Pair64 warp_sums[kPlanThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int64_t r_begin = static_cast<int64_t>(blockIdx.x) * p.rows_per_cta;
  const int64_t r_end = min(p.n_rows, r_begin + p.rows_per_cta);
  const uint32_t page_size = static_cast<uint32_t>(p.page_size);
  const bool lead = blockIdx.x == 0;
  Pair64 base{0, 0};
  int64_t taken = 0;
  for (int64_t s0 = 0; s0 < p.n_seqs; s0 += kChunk) {
    if (!lead && base.rows >= r_end) break;
    int32_t cached[kPerThread], fresh[kPerThread];
    SeqNeed n[kPerThread];
    Pair64 mine{0, 0};
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int64_t s = s0 + tid * kPerThread + i;
      cached[i] = s < p.n_seqs ? p.cached[s] : 0;
      fresh[i] = s < p.n_seqs ? p.fresh[s] : 0;
    }
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      n[i] = seq_need_upto(cached[i], fresh[i], p.page_size, p.most);
      mine = mine + Pair64{n[i].rows, n[i].need};
    }
    Pair64 total;
    Pair64 at = base + block_prefix(mine, warp_sums, total);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int64_t s = s0 + tid * kPerThread + i;
      const int x = tid * kPerThread + i;
      const bool served = seq_served(n[i], at.need, p.n_free);
      row0[x] = static_cast<int32_t>(min(at.rows, p.n_rows));
      page0[x] = served ? static_cast<int32_t>(min(at.need, p.n_free)) : -1;
      have_s[x] = static_cast<int32_t>(n[i].have);
      cached_s[x] = cached[i];
      if (lead && s < p.n_seqs) {
        if (!served) record_error(p.checks, n[i].valid ? EFG_ENOMEM : EFG_EINVAL);
        p.cu[s] = static_cast<int32_t>(min(at.rows, p.n_rows));
        p.kv_len[s] = served ? cached[i] + fresh[i] : 0;
        if (s == p.n_seqs - 1) {
          if (at.rows + n[i].rows > p.n_rows) record_error(p.checks, EFG_EINVAL);
          p.cu[p.n_seqs] = static_cast<int32_t>(min(at.rows + n[i].rows, p.n_rows));
        }
      }
      // pages taken: the end of the last need that is served (they are contiguous from 0)
      taken = max(taken, served && n[i].need ? at.need + n[i].need : 0);
      at = at + Pair64{n[i].rows, n[i].need};
    }
    __syncthreads();
    const int count = static_cast<int>(min(static_cast<int64_t>(kChunk), p.n_seqs - s0));
    const int64_t lo = max(r_begin, base.rows), hi = min(r_end, base.rows + total.rows);
    for (int64_t r = lo + tid; r < hi; r += kPlanThreads) {
      int a = 0, b = count;  // largest i with row0[i] <= r
      while (b - a > 1) {
        const int m = (a + b) / 2;
        if (row0[m] <= r)
          a = m;
        else
          b = m;
      }
      int32_t slot = -1, pos = -1;
      if (page0[a] >= 0) {
        // (a served sequence's positions fit 32 bits)
        const uint32_t at_pos = static_cast<uint32_t>(cached_s[a]) + static_cast<uint32_t>(r - row0[a]);
        const uint32_t pi = at_pos / page_size, off = at_pos - pi * page_size;
        int32_t* entry = p.table + (s0 + a) * p.max_pages + pi;
        const bool old = pi < static_cast<uint32_t>(have_s[a]);
        const int32_t page = old ? *entry : p.free[page0[a] + (pi - static_cast<uint32_t>(have_s[a]))];
        if (page_ok(page, p.n_pages)) {
          slot = static_cast<int32_t>(page * p.page_size + off);
          pos = static_cast<int32_t>(at_pos);
        } else {
          record_error(p.checks, EFG_EINVAL);
        }
        if (!old && off == 0) *entry = page;
      }
      p.slots[r] = slot;
      p.positions[r] = pos;
    }
    base = base + total;
    __syncthreads();  // the shared arrays are rewritten by the next chunk
  }
  // rows behind the last sequence
  for (int64_t r = max(r_begin, base.rows) + tid; r < r_end; r += kPlanThreads) p.slots[r] = p.positions[r] = -1;
  if (lead) {
    for (int o = 16; o > 0; o >>= 1) taken = max(taken, static_cast<int64_t>(__shfl_xor_sync(0xFFFFFFFFu, taken, o)));
    if ((tid & 31) == 0) warp_sums[tid >> 5].need = taken;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kPlanThreads / 32; ++w) taken = max(taken, warp_sums[w].need);
      *p.taken = static_cast<int32_t>(taken);
      if (p.n_seqs == 0) p.cu[0] = 0;
    }
  }
}

// ---------------------------------------------------------------- rotated store
struct StoreParams {
  void *q_out, *k_cache, *v_cache;
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  const int32_t *slots, *positions;
  const float *cos, *sin;  // null: no rotation
  int64_t n_slots, max_pos;
  int heads, kv_heads, head_dim;
  int* checks;
};

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half narrow<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// One CTA column per row, one thread per pair of V-wide pieces at dims i and i + head_dim / 2 of
// one head (the two halves that a half-split rotation mixes, src/kernels.cpp:133-147); value
// heads take the same shape without the rotation. The rotation is the decoder's: products and
// sums rounded one by one in FP32, then once to the cache's type. Bound by HBM: 178 MB (prompts up to 4096 FP32
// tokens, 32 query and 2 x 8 heads of 128, to BF16 pages) in 30.6 us, 5.8 TB/s; of few rows by latency.
template <typename Tin, typename Tout, int V>
__global__ void __launch_bounds__(256) page_store_kernel(const StoreParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int half = p.head_dim / 2, per_head = half / V;
  const int e = blockIdx.y * blockDim.x + threadIdx.x;
  const int qh = p.q ? p.heads : 0;
  if (e >= (qh + 2 * p.kv_heads) * per_head) return;
  const int64_t row = blockIdx.x;
  const int head = e / per_head, i = (e - head * per_head) * V;
  const int32_t slot = p.slots[row], pos = p.positions[row];
  const bool is_q = head < qh, is_k = !is_q && head < qh + p.kv_heads;
  if (pos < 0 || (!is_q && slot < 0)) return;  // a padding row: everything of it stays as it was
  if (slot >= p.n_slots || pos >= p.max_pos) {
    record_error(p.checks, EFG_EINVAL);
    return;
  }
  const int kvh = head - qh - (is_k ? 0 : p.kv_heads);
  const Tin* src = is_q   ? static_cast<const Tin*>(p.q) + row * p.q_stride + head * p.head_dim
                   : is_k ? static_cast<const Tin*>(p.k) + row * p.k_stride + kvh * p.head_dim
                          : static_cast<const Tin*>(p.v) + row * p.v_stride + kvh * p.head_dim;
  Tout* dst = is_q ? static_cast<Tout*>(p.q_out) + (row * p.heads + head) * p.head_dim
                   : static_cast<Tout*>(is_k ? p.k_cache : p.v_cache) +
                         (static_cast<int64_t>(slot) * p.kv_heads + kvh) * p.head_dim;
  const Vec<Tin, V> a = *reinterpret_cast<const Vec<Tin, V>*>(src + i);
  const Vec<Tin, V> b = *reinterpret_cast<const Vec<Tin, V>*>(src + i + half);
  Vec<Tout, V> x, y;
  if (p.cos && (is_q || is_k)) {
    const Vec<float, V> c = *reinterpret_cast<const Vec<float, V>*>(p.cos + static_cast<int64_t>(pos) * half + i);
    const Vec<float, V> s = *reinterpret_cast<const Vec<float, V>*>(p.sin + static_cast<int64_t>(pos) * half + i);
#pragma unroll
    for (int t = 0; t < V; ++t) {
      const float fa = widen(a.v[t]), fb = widen(b.v[t]);
      x.v[t] = narrow<Tout>(__fsub_rn(__fmul_rn(fa, c.v[t]), __fmul_rn(fb, s.v[t])));
      y.v[t] = narrow<Tout>(__fadd_rn(__fmul_rn(fb, c.v[t]), __fmul_rn(fa, s.v[t])));
    }
  } else {
#pragma unroll
    for (int t = 0; t < V; ++t) {
      x.v[t] = narrow<Tout>(widen(a.v[t]));
      y.v[t] = narrow<Tout>(widen(b.v[t]));
    }
  }
  *reinterpret_cast<Vec<Tout, V>*>(dst + i) = x;
  *reinterpret_cast<Vec<Tout, V>*>(dst + i + half) = y;
}

// A launch whose start overlaps the end of the kernel before it (both kernels wait for that one's results first).
template <typename P>
int launch_chained(void (*fn)(const P), dim3 grid, int threads, const P& p, cudaStream_t s, const char* what) {
  cudaLaunchConfig_t cf{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cf.gridDim = grid;
  cf.blockDim = dim3(static_cast<unsigned>(threads));
  cf.stream = s;
  cf.attrs = attr;
  cf.numAttrs = 1;
  EFG_TRY_CUDA(cudaLaunchKernelEx(&cf, fn, p), what);
  return EFG_OK;
}

template <typename Tin, typename Tout>
int store_rows(const StoreParams& p, size_t n_rows, int V, cudaStream_t s) {
  const int qh = p.q ? p.heads : 0, items = (qh + 2 * p.kv_heads) * (p.head_dim / 2 / V);
  const int threads = std::min(256, (items + 31) / 32 * 32);
  const dim3 grid(static_cast<unsigned>(n_rows), static_cast<unsigned>((items + threads - 1) / threads));
  return launch_chained(V == 4 ? page_store_kernel<Tin, Tout, 4> : page_store_kernel<Tin, Tout, 1>, grid, threads, p, s,
                        "page_store launch");
}

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace
}  // namespace efg

using efg::fail;

extern "C" {

int efg_page_plan(const efg_page_plan_args* args, void* stream) {
  if (!args) return fail(EFG_EINVAL, "page_plan: null pointer");
  const auto& [d_block_table, max_pages, d_slots, d_positions, n_rows, d_cu, d_kv_len, d_taken, d_cached, d_new, n_seqs,
               d_free, n_free, n_pages, page_size] = *args;
  if (!d_cu || !d_taken || (n_rows && (!d_slots || !d_positions)) || (n_free && !d_free) ||
      (n_seqs && (!d_kv_len || !d_cached || !d_new || (max_pages && !d_block_table))))
    return fail(EFG_EINVAL, "page_plan: null pointer");
  if (page_size == 0 || page_size > (1u << 30)) return fail(EFG_EINVAL, "page_plan: page size %zu", page_size);
  if (n_pages > 0x7FFFFFFFull / page_size)
    return fail(EFG_EINVAL, "page_plan: %zu pages of %zu slots pass the 2^31 slots of a cache", n_pages, page_size);
  if (n_rows > 0x7FFFFFFFull || n_seqs > (1ull << 24) || n_free > 0x7FFFFFFFull || max_pages > 0x7FFFFFFFull)
    return fail(EFG_EINVAL, "page_plan: a size is out of range");
  const struct {
    const void* at;
    size_t n;
  } parts[] = {{d_block_table, n_seqs * max_pages}, {d_slots, n_rows}, {d_positions, n_rows}, {d_cu, n_seqs + 1},
               {d_kv_len, n_seqs}, {d_taken, 1}, {d_cached, n_seqs}, {d_new, n_seqs}, {d_free, n_free}};
  for (int i = 0; i < 6; ++i)  // the outputs, against everything behind them
    for (int j = i + 1; j < 9; ++j)
      if (efg::overlap(parts[i].at, parts[i].n * 4, parts[j].at, parts[j].n ? 1 : 0, 0, parts[j].n, 4))
        return fail(EFG_EINVAL, "page_plan: an output overlaps an input or another output");
  efg::DeviceInfo* dev = efg::current_device();
  if (!dev) return EFG_ECUDA;
  efg::PlanParams p{};
  p.table = d_block_table;
  p.slots = d_slots;
  p.positions = d_positions;
  p.cu = d_cu;
  p.kv_len = d_kv_len;
  p.taken = d_taken;
  p.cached = d_cached;
  p.fresh = d_new;
  p.free = d_free;
  p.max_pages = static_cast<int64_t>(max_pages);
  p.n_rows = static_cast<int64_t>(n_rows);
  p.n_seqs = static_cast<int64_t>(n_seqs);
  p.n_free = static_cast<int64_t>(n_free);
  p.n_pages = static_cast<int64_t>(n_pages);
  p.page_size = static_cast<int64_t>(page_size);
  p.most = efg::most_positions(p.max_pages, p.page_size);
  p.checks = dev->d_checks;
  const size_t ctas = std::max<size_t>(1, std::min<size_t>(dev->sm_count, (n_rows + 511) / 512));
  p.rows_per_cta = static_cast<int64_t>((n_rows + ctas - 1) / ctas);
  return efg::launch_chained(efg::page_plan_kernel, dim3(static_cast<unsigned>(ctas)), efg::kPlanThreads, p,
                             static_cast<cudaStream_t>(stream), "page_plan launch");
}

int efg_page_store(const efg_page_store_args* args, void* stream) {
  if (!args) return fail(EFG_EINVAL, "page_store: null pointer");
  const auto& [type, cache_type, d_q_out, d_k_cache, d_v_cache, n_slots, d_q, q_stride, d_k, k_stride, d_v, v_stride,
               d_slots, d_positions, n_rows, d_cos, d_sin, max_pos, heads, kv_heads, head_dim] = *args;
  if (type < EFG_F32 || type > EFG_BF16) return fail(EFG_EINVAL, "page_store: unknown type %d", type);
  if (cache_type != type && (type != EFG_F32 || cache_type < EFG_F32 || cache_type > EFG_BF16))
    return fail(EFG_EINVAL, "page_store: the cache has the rows' type, or F16 or BF16 for F32 rows (got %d for %d)",
                cache_type, type);
  if (head_dim == 0 || head_dim % 2 || head_dim > 256)
    return fail(EFG_EINVAL, "page_store: head_dim %zu is not an even number up to 256", head_dim);
  if (kv_heads == 0 || kv_heads > 4096 || (d_q && (heads == 0 || heads > 4096)))
    return fail(EFG_EINVAL, "page_store: %zu query and %zu key heads", heads, kv_heads);
  if (n_rows > 0x7FFFFFFFull || n_slots > 0x7FFFFFFFull || max_pos > 0x7FFFFFFFull)
    return fail(EFG_EINVAL, "page_store: a size is out of range");
  if ((d_q != nullptr) != (d_q_out != nullptr) || (d_cos != nullptr) != (d_sin != nullptr))
    return fail(EFG_EINVAL, "page_store: q and q_out, and cos and sin, come together");
  if (n_rows == 0) return EFG_OK;
  if (!d_k || !d_v || !d_k_cache || !d_v_cache || !d_slots || !d_positions)
    return fail(EFG_EINVAL, "page_store: null pointer");
  if ((d_q && q_stride < heads * head_dim) || k_stride < kv_heads * head_dim || v_stride < kv_heads * head_dim)
    return fail(EFG_EINVAL, "page_store: a row stride is shorter than a row");
  const size_t es = type == EFG_F32 ? 4 : 2, co = cache_type == EFG_F32 ? 4 : 2;
  const size_t q_row = heads * head_dim, kv_row = kv_heads * head_dim;
  const bool in_place = d_q == d_q_out && type == cache_type && q_stride == q_row;
  auto meets = [&](const void* out, size_t n_out, bool own_q) {
    return (!own_q && efg::overlap(out, n_out, d_q, n_rows, q_stride, q_row, es)) ||
           efg::overlap(out, n_out, d_k, n_rows, k_stride, kv_row, es) ||
           efg::overlap(out, n_out, d_v, n_rows, v_stride, kv_row, es) ||
           efg::overlap(out, n_out, d_slots, 1, 0, n_rows, 4) || efg::overlap(out, n_out, d_positions, 1, 0, n_rows, 4) ||
           efg::overlap(out, n_out, d_cos, 1, 0, max_pos * (head_dim / 2), 4) ||
           efg::overlap(out, n_out, d_sin, 1, 0, max_pos * (head_dim / 2), 4);
  };
  const size_t cache = n_slots * kv_row * co;
  if (meets(d_q_out, n_rows * q_row * co, in_place) || meets(d_k_cache, cache, false) || meets(d_v_cache, cache, false))
    return fail(EFG_EINVAL, "page_store: an output overlaps an input");
  if (efg::overlap(d_k_cache, cache, d_v_cache, n_slots, kv_row, kv_row, co) ||
      efg::overlap(d_q_out, n_rows * q_row * co, d_k_cache, n_slots, kv_row, kv_row, co) ||
      efg::overlap(d_q_out, n_rows * q_row * co, d_v_cache, n_slots, kv_row, kv_row, co))
    return fail(EFG_EINVAL, "page_store: outputs overlap");
  efg::DeviceInfo* dev = efg::current_device();
  if (!dev) return EFG_ECUDA;
  efg::StoreParams p{};
  p.q_out = d_q_out;
  p.k_cache = d_k_cache;
  p.v_cache = d_v_cache;
  p.q = d_q;
  p.k = d_k;
  p.v = d_v;
  p.q_stride = static_cast<int64_t>(q_stride);
  p.k_stride = static_cast<int64_t>(k_stride);
  p.v_stride = static_cast<int64_t>(v_stride);
  p.slots = d_slots;
  p.positions = d_positions;
  p.cos = d_cos;
  p.sin = d_sin;
  p.n_slots = static_cast<int64_t>(n_slots);
  p.max_pos = d_cos ? static_cast<int64_t>(max_pos) : 0x7FFFFFFFll;
  p.heads = static_cast<int>(heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.head_dim = static_cast<int>(head_dim);
  p.checks = dev->d_checks;
  const bool wide = head_dim % 8 == 0 && q_stride % 4 == 0 && k_stride % 4 == 0 && v_stride % 4 == 0 &&
                    efg::aligned(d_q, 4 * es) && efg::aligned(d_k, 4 * es) && efg::aligned(d_v, 4 * es) &&
                    efg::aligned(d_q_out, 4 * co) && efg::aligned(d_k_cache, 4 * co) &&
                    efg::aligned(d_v_cache, 4 * co) && efg::aligned(d_cos, 16) && efg::aligned(d_sin, 16);
  const int V = wide ? 4 : 1;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (type == EFG_F16) return efg::store_rows<__half, __half>(p, n_rows, V, s);
  if (type == EFG_BF16) return efg::store_rows<__nv_bfloat16, __nv_bfloat16>(p, n_rows, V, s);
  if (cache_type == EFG_F16) return efg::store_rows<float, __half>(p, n_rows, V, s);
  if (cache_type == EFG_BF16) return efg::store_rows<float, __nv_bfloat16>(p, n_rows, V, s);
  return efg::store_rows<float, float>(p, n_rows, V, s);
}

}  // extern "C"
