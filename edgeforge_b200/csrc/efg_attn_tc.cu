// efg_attn_tc.cu - attention of large row tiles (prompts, chunks) on the 5th-generation tensor cores: 16-bit types
// to head size 128, F32 to 64.
//
// One CTA per SM owns two 128-row tiles of one key head, each of floor(128 / group) tokens times the
// group's query heads (row = token * group + head), so a group shares its keys and the two tiles share
// every key and value tile (128 positions) that TMA brings into a ring. Per tile of keys and row tile:
//   S = Q K^T       tcgen05.mma, Q and K from shared memory, S (FP32) in TMEM;
//   P = 2^(S - ref) one softmax thread per row: TMEM -> 128 registers -> exponentials -> 16-bit P back
//                   into TMEM;
//   O += P V        tcgen05.mma with A = P from TMEM, O (FP32) in TMEM.
// The two row tiles alternate: while one is in its softmax, the tensor cores work for the other.
// The reference value ref follows the running maximum lazily: it moves (and O is multiplied) only when
// the maximum has grown by more than 2^8, so weights stay below 256 and O is touched rarely.
//
// What bounds it: at head size 128 the two products of a 128 x 128 tile take 1024 tensor-core cycles and
// its 16384 exponentials 1024 cycles of the special function units, so neither may wait for the other;
// at 64 the exponentials (and the instructions around them) are the bound. Measured: one 8192-token
// prompt, 32 query and 8 key heads of 128, BF16: 550-565 us, 970-1000 TFLOP/s, in a run of seconds, where the clock
// drops at the power cap; 480 us, 1145 TFLOP/s, in one of milliseconds, the tensor pipe and the exponentials' pipe busy
// for 54 % each. P is rounded to the inputs' type, because A and B of an MMA have one type: a second
// product for what that leaves out would take half of the tensor cores' time again. Error of that prompt's rows against
// 64 bits 2.2e-3, of FP32 weights 1.7e-3 (the output's own rounding). Measured and not kept: a part of the
// exponentials as a degree-4 polynomial on the FMA pipes (no gain at any share), turns at the
// exponentials for the two warps of a scheduler (491 against 430 us at 64: one warp alone does not fill
// the special function units), sums and packing one quarter behind the exponentials (540 against 486).
//
// Roles (12 warps): 0-3 and 4-7 softmax and epilogue of row tiles 0 and 1, 8 TMA, 9 (and 11) MMA, 10 scheduler: a CTA
// walks many pairs of row tiles, and loads and products of the next one run during the epilogue of the
// one before. (Registers: 2 x 128 x 224 for the softmax, 128 x 56 for the other warpgroup, of the launch's
// 384 x 168.) TMEM (512 columns): S0 | S1 | O0 | O1, at head size 64 then P0 | P1: the next S is there before
// the softmax asks for it. At 128 P overwrites S, and the other row tile's work fills the wait. With a workspace
// (paged chunks) the work is one line of key tiles cut into equal runs, and a second launch joins the
// rows of items that were cut, in order.
//
// F32 (16 warps; registers 2 x 128 x 160 and 2 x 128 x 96 of 512 x 128): TMA brings FP32 tiles, four converter warps
// (12-15) turn each into two F16 tiles hi + lo, scaled by a power of two (keys: one for the tile, values: one for each
// dim), and S = Qh Kh + Qh Kl + Ql Kh, O = Ph [Vh | Vl] + Pl Vh in the same instructions, with P split as well. O of each
// key tile begins at zero and is added up in the softmax threads' registers, in FP32. Bound by the converters and by
// what spills to local memory (L1 is all shared memory here): S is read 32 columns at a time in loops that stay loops
// (unrolled: 131 us), without the columns that no row of a warp sees (23 tokens 14.4 -> 13.1 us). 2048 tokens, 32 query
// and 4 key heads of 64: 118-123 us (in TF32 parts on the warp-level tensor cores: 436); error of a row 4.4e-7.
#include <algorithm>

#include <cuda_runtime.h>

#include "efg_attn.cuh"
#include "efg_attn_launch.h"
#include "efg_host.h"
#include "efg_tcgen05.cuh"

namespace efg {
namespace {

constexpr int kTileKeys = 128, kTileRows = 128;
template <typename T>
constexpr bool is_f32 = std::is_same_v<T, float>;
template <typename T>
constexpr int threads = is_f32<T> ? 512 : 384;
constexpr uint32_t kPanel = 128 * 128;  // 128 rows of 64 16-bit values, 128-byte swizzled
// Powers of two that the maximum may grow before O is rescaled; F32 weights are held 2^12 higher, so that both
// their F16 parts stay in range and small ones keep their digits.
template <typename T>
constexpr float kLazy = is_f32<T> ? 3.f : 8.f;
constexpr int kRaise = 12;

// Panels of an operand tile (a row of 64 16-bit values each): the head's dims, or the hi and the lo part of 64 FP32
// dims; operand stages, and stages of FP32 tiles on their way to the converters.
template <typename T, int D>
constexpr int panels = is_f32<T> ? 2 : D / 64;
template <typename T, int D>
constexpr int kv_stages = is_f32<T> ? 3 : D == 64 ? 8 : 5;
template <typename T>
constexpr int staging = is_f32<T> ? 2 : 0;
template <typename T, int D>
constexpr size_t smem_bytes = 1024 + static_cast<size_t>(2 + kv_stages<T, D> + staging<T>) * panels<T, D> * kPanel;

// A value tile as the B operand of O += P V: keys run along K, so the tile (rows of keys, 64 dims of 128
// bytes, 128-byte swizzle) is MN-major: 64-dim panels kPanel apart, groups of 8 keys 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_values(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(kPanel >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Instruction descriptor: FP32 accumulator, A and B F16 or BF16, A K-major, B K-major or MN-major.
template <typename T>
constexpr uint32_t idesc_of(uint32_t N, bool b_mn) {
  const uint32_t fmt = std::is_same_v<T, __nv_bfloat16> ? 1u : 0u;  // (F32: two F16 parts)
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

// Largest and least of three magnitudes (NaN left out).
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float min3_abs(float a, float b, float c) {
  float r;
  asm("min.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Ties the registers of a TMEM load to the point after its wait.
__device__ __forceinline__ void after_wait(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]),
                 "+r"(r[i + 6]), "+r"(r[i + 7]));
}

// Weights of 32 columns, packed to 16 bits; `total` collects the unrounded weights. Masked places (-inf) come
// out as exact zeros.
template <typename T>
__device__ __forceinline__ void weights32(const uint32_t* s, uint64_t scale, uint64_t nref, uint64_t (&total)[2],
                                          uint32_t (&out)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float a, b;
    unpair(fma2(pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale, nref), a, b);
    a = ex2(a);
    b = ex2(b);
    total[i % 2] = add2(total[i % 2], pair(a, b));
    out[i] = pack2<T>(a, b);
  }
}

// The lo parts of weights and values are held 2^11 times larger than they are: next to their hi part that is the
// largest factor that F16 takes, and it keeps the digits of what lies up to 2^28 below the largest.
constexpr float kLoUp = 2048.f;

// The same for F32: each weight (below 2^3, raised by 2^12) as hi + 2^-11 lo in F16, within 2^-22 of itself or 2^-48 of 1.
__device__ __forceinline__ void weights32_split(const uint32_t* s, uint64_t scale, uint64_t nref, uint64_t (&total)[2],
                                                uint32_t (&hi)[16], uint32_t (&lo)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float a, b;
    unpair(fma2(pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale, nref), a, b);
    // (raised by a product, not in the exponent: next to 0 that keeps more of its digits)
    constexpr float kUp = static_cast<float>(1 << kRaise);
    const uint64_t w = fma2(pair(ex2(a), ex2(b)), pair(kUp, kUp), 0);
    total[i % 2] = add2(total[i % 2], w);
    unpair(w, a, b);
    const __half2 h = __floats2half2_rn(a, b);
    const float2 back = __half22float2(h);
    hi[i] = *reinterpret_cast<const uint32_t*>(&h);
    const uint64_t rest = fma2(pair(back.x, back.y), pair(-1.f, -1.f), w);  // exact
    unpair(fma2(rest, pair(kLoUp, kLoUp), 0), a, b);
    lo[i] = pack2<__half>(a, b);
  }
}

// Four FP32 values, scaled by powers of two, as F16 parts hi + lo, or hi + lo / kLoUp: within 2^-22 of the value or
// 2^-25 (2^-36) of the scaled unit.
template <bool kUp>
__device__ __forceinline__ void split4(const float4& x, const float4& scale, uint2& hi, uint2& lo) {
  const auto split2 = [](uint64_t v, uint32_t& hi, uint32_t& lo) {
    float a, b;
    unpair(v, a, b);
    const __half2 h = __floats2half2_rn(a, b);
    const float2 back = __half22float2(h);
    uint64_t rest = fma2(pair(back.x, back.y), pair(-1.f, -1.f), v);  // exact
    if (kUp) rest = fma2(rest, pair(kLoUp, kLoUp), 0);
    unpair(rest, a, b);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack2<__half>(a, b);
  };
  split2(fma2(pair(x.x, x.y), pair(scale.x, scale.y), 0), hi.x, lo.x);
  split2(fma2(pair(x.z, x.w), pair(scale.z, scale.w), 0), hi.y, lo.y);
}
// Largest finite magnitude of a quad and what came before.
__device__ __forceinline__ float finite_max(float m, const float4& v) {
  const float a[4] = {fabsf(v.x), fabsf(v.y), fabsf(v.z), fabsf(v.w)};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = a[i] <= 3.402823466e38f ? fmaxf(m, a[i]) : m;
  return m;
}
// Exponent of the largest magnitude (held at -100 and above), and 2^e.
__device__ __forceinline__ int exponent_of(float m) { return max(static_cast<int>(__float_as_uint(m) >> 23) - 127, -100); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
constexpr int kTop = 14;  // split operands are scaled so that their largest value is below 2^(kTop + 1)
// A value that is far larger than the rest of what shares its scale (also one at a position that a row does not see, or
// that it gives next to no weight) takes digits from the rest.
//   Keys: one scale for a tile. A score loses up to 2^-31 scale 2^(eq + ek) (eq, ek: exponents of the query and of the
// largest key); rows where that passes 2^-15 are computed again in FP32 (attend_row).
//   Values: a scale for every dim of a tile. A weighted sum loses up to 2^(ev - 50) of the sum of the weights, and
// 2^(ev - 48) for every key that weighs less than 2^-26 (ev: exponent of the dim's largest value). Where every value of
// the dim is zero or at least 2^(ev - 26), the first is below 2^-24 of sum w |v|, whatever the weights are. Where one is
// not, rows with a sum below 2^(ev - 26) of the weights' are computed again: of normally distributed values a dim in
// a thousand tiles, and then one row in ten thousand. (kTop + kRaise = 26: a dim's unit is that bound.) The second is
// left where the keys that weigh more have zeros in the dim: to look at these rows too costs 3 to 11 % without any zero.
constexpr float kScoreRange = 65536.f;

// Whether `ok` holds for all 128 converter threads; a barrier among them.
__device__ __forceinline__ bool all_converters(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(ok ? 1u : 0u)
      : "memory");
  return r != 0;
}

// All threads of the CTA, from inside their roles.
template <int kThreads>
__device__ __forceinline__ void cta_barrier() {
  __syncwarp();
  asm volatile("bar.sync 0, %0;" ::"n"(kThreads) : "memory");
}

// Asks the hardware for a CTA of this grid that has not started: its place is taken over by this CTA
// (cluster launch control). The answer, 16 bytes, completes on `bar`.
__device__ __forceinline__ void ask_next_cta(uint4* answer, uint64_t* bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
          smem_addr(answer)),
      "r"(smem_addr(bar))
      : "memory");
}
// The taken CTA's blockIdx.x, or -1 when every CTA has started (nothing may be asked for after that).
__device__ __forceinline__ int next_cta(const uint4* answer) {
  uint32_t got, x, y, z;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 a;\n\t"
      "ld.shared.b128 a, [%4];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, %2, %3, _}, a;\n\t}"
      : "=&r"(got), "=&r"(x), "=&r"(y), "=&r"(z)
      : "r"(smem_addr(answer))
      : "memory");
  return got ? static_cast<int>(x) : -1;
}

// An item that is cut along its keys: its pieces are slot `first` of CTA i (1: the last part of its run, 0: all
// of it) and slot 0 of the CTAs behind it.
struct alignas(16) TcJoin {
  Chunk c;
  int32_t kvh, token0, first, parts;  // parts 0: nothing begins here that is cut
};

// 32 columns of O; F32: the products of both hi parts plus, 64 columns on, those with a lo part.
template <bool kF32>
__device__ __forceinline__ void load_o(uint32_t addr, uint32_t (&o)[32]) {
  tmem_ld32(addr, o);
  if constexpr (kF32) {
    uint32_t lo[32];
    tmem_ld32(addr + 64, lo);
    tmem_wait_ld();
    after_wait(o);
    after_wait(lo);
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      float a, b;
      unpair(fma2(pair(__uint_as_float(lo[e]), __uint_as_float(lo[e + 1])), pair(1.f / kLoUp, 1.f / kLoUp),
                  pair(__uint_as_float(o[e]), __uint_as_float(o[e + 1]))), a, b);
      o[e] = __float_as_uint(a);
      o[e + 1] = __float_as_uint(b);
    }
  } else {
    tmem_wait_ld();
    after_wait(o);
  }
}

struct TcParams {
  AttnParams a;
  TcJoin* joins;      // [ctas]; null: whole items, handed out by the hardware
  float* slots;       // [ctas][2]{top[256], sum[256], o[D / 4][256][4]}
  int tokens;         // tokens of a row tile
  int tiles;          // pairs of row tiles of one key head, some of which may turn out to be empty
  int tiles_per_seq;  // of them at fixed places for every sequence, or 0: found by a scan
  int box_rows;       // rows of one key / value box
};

// What the begin and end of an item cost, in key tiles, and the weight of a run, at least: not sharp. Chunks of 64 to 512
// BF16 rows over 2000 to 65536 positions, alone and beside 255 single tokens, take the same within the noise (3 %) with a
// cost of 1 or 6, and with runs of 2 or 8.
constexpr int kItemCost = 3, kMinRun = 4;

// A pair of row tiles of one key head, or a run of its key tiles, as the scheduler warp hands it to the roles.
struct Item {
  Chunk c;
  int32_t kvh, token0;
  int32_t first, count;  // key tiles
  int32_t slot;          // -1: all of them, the rows are written out; else the workspace slot of this CTA
  int32_t stop;
};

// What a role derives from an item: tokens of the two row tiles, the keys that the last one sees, and how many
// of the item's key tiles row tile i uses.
struct Plan {
  int tok[2], n[2], see_all;
};
__device__ __forceinline__ int keys_of(const Chunk& c, int token_end) { return seen_by(c, c.begin + token_end - 1); }
__device__ __forceinline__ Plan plan_of(const Item& w, int tokens) {
  Plan a;
  a.see_all = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    a.tok[i] = max(0, min(tokens, w.c.end - w.c.begin - w.token0 - i * tokens));
    const int last = a.tok[i] ? keys_of(w.c, w.token0 + i * tokens + a.tok[i]) : 0;
    a.see_all = max(a.see_all, last);
    a.n[i] = max(0, min(w.first + w.count, (last + kTileKeys - 1) / kTileKeys) - w.first);
  }
  return a;
}
// Key tiles of the pair of row tiles that begins at token0.
__device__ __forceinline__ int tiles_of_pair(const Chunk& c, int token0, int pair_tokens) {
  return (keys_of(c, min(c.end - c.begin, token0 + pair_tokens)) + kTileKeys - 1) / kTileKeys;
}
// Weight of a sequence under one key head: of each pair its begin and end, then its key tiles.
__device__ __forceinline__ int weight_of(const AttnParams& p, int64_t seq, int pair_tokens) {
  Chunk c;
  if (!chunk_of_seq(p, seq, c)) return 0;
  int sum = 0;
  for (int t = 0; t < c.end - c.begin; t += pair_tokens) sum += kItemCost + tiles_of_pair(c, t, pair_tokens);
  return sum;
}

// kRuns: the work is cut into runs (tp.joins and tp.slots are set); otherwise whole items are handed out. Apart,
// because the code of one costs the other: one 8192-token prompt takes 512 us with both in one kernel, 490
// without the runs.
template <typename T, int D, bool kRuns>
__global__ void __launch_bounds__(threads<T>, 1)
    attn_tc_kernel(const __grid_constant__ TcParams tp, const __grid_constant__ CUtensorMap map_q,
                   const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  constexpr bool kF32 = is_f32<T>;
  using E = std::conditional_t<kF32, __half, T>;  // of the MMA operands
  constexpr int kThreads = threads<T>, kPanels = panels<T, D>, kStages = kv_stages<T, D>, kStaging = kF32 ? 2 : 1;
  // P beside S in TMEM: the next S does not wait for the value product
  constexpr bool kApart = !kF32 && D == 64;
  constexpr uint32_t kTileBytes = kPanels * kPanel;
  // columns of O per row tile (F32: products with V hi, then with V lo), where P lies
  constexpr uint32_t kColO = 256, kWideO = kF32 ? 128 : D, kColP = kApart ? 384 : 0, kStepP = kApart ? 64 : 128;
  static_assert(!kF32 || D == 64);
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t q_full, q_empty, kv_full[kStages], kv_empty[kStages], s_full[2], s_free[2], p_ready[2], pv_done[2],
      drained[2], item_full[2], item_empty[2], fetch, asked;
  __shared__ uint64_t stage_full[kStaging], stage_empty[kStaging], exp_full[8];
  // exponents of the split key tiles, by ring item; units of the value tiles' dims (what 1 of O stands for), by value
  // tile; by item with keys the biased exponent of the largest unit of every dim, 0 where its values are close enough;
  // by dim the exponents of each warp's largest and least values, a byte each
  __shared__ int exp_s[8];
  __shared__ float4 unit_s[kF32 ? 3 : 1][16];
  __shared__ uint4 wide_s[2][kF32 ? 4 : 1], dims_s[2][kF32 ? 16 : 1];
  __shared__ float max_s[2][4];
  __shared__ uint4 answer;
  __shared__ int run_s[5];
  int* scan_s = reinterpret_cast<int*>(unit_s);  // (before the roles begin)
  __shared__ Item items[2];
  __shared__ uint32_t tmem_slot;
  __shared__ uint64_t until_s;  // waits go on until then (wait_own)
  const AttnParams& p = tp.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t raw = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* q_s = smem_raw + (base - raw);
  uint8_t* ring = q_s + 2 * kTileBytes;
  uint8_t* stage = ring + kStages * kTileBytes;
  if (tid == 0) {
    mbar_init(&q_full, kF32 ? 256 : 1);
    mbar_init(&q_empty, kApart ? 2 : 1);
    mbar_init(&fetch, 1);
    mbar_init(&asked, 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&kv_full[i], kF32 ? 128 : 1);
      mbar_init(&kv_empty[i], kApart ? 2 : 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 128);
      mbar_init(&p_ready[i], 128);
      mbar_init(&pv_done[i], 1);
      mbar_init(&item_full[i], 1);
      // 8 softmax warps (when they are done with it), TMA, MMA, converters
      mbar_init(&item_empty[i], kApart ? 11 : kF32 ? 14 : 10);
      mbar_init(&drained[i], 1);
    }
    for (int i = 0; i < kStaging; ++i) {
      mbar_init(&stage_full[i], 1);
      mbar_init(&stage_empty[i], 128);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&exp_full[i], 1);
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(&tmem_slot, 512);
  // (the next launch may not begin early: its CTAs would take SMs from items that are still to be handed out, 120
  // against 127 us for 2048 FP32 tokens call after call)
  pdl_wait();
  if (tid == 0) move_on(&until_s);
  if (!kRuns && tp.tiles_per_seq == 0 && blockIdx.x == 0) check_offsets(p);
  if constexpr (kRuns) {
    // This CTA's run of the line of all items' key tiles: every thread adds up a block of sequences, the one
    // whose block holds the beginning finds the sequence.
    const int n_seqs = static_cast<int>(p.n_seqs), per = (n_seqs + kThreads - 1) / kThreads;
    const int s_lo = min(n_seqs, tid * per), s_hi = min(n_seqs, s_lo + per), pair_tokens = 2 * tp.tokens;
    int mine = 0;
    for (int x = s_lo; x < s_hi; ++x) mine += weight_of(p, x, pair_tokens) * p.kv_heads;
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
    for (int x = 0; x < kThreads / 32; ++x) {
      if (x < warp) before += scan_s[x];
      line += scan_s[x];
    }
    const int n_runs = min(static_cast<int>(gridDim.x), max(1, line / kMinRun));
    if (tid == 0) {
      tp.joins[blockIdx.x].parts = 0;
      run_s[2] = line;
      run_s[3] = n_runs;
    }
    if (line > 0 && static_cast<int>(blockIdx.x) < n_runs) {
      const Runs runs(line, n_runs);
      const int begin = static_cast<int>(runs.begin(blockIdx.x));
      if (begin >= before && begin < before + mine) {
        int at = begin - before, x = s_lo;
        for (int n; (n = weight_of(p, x, pair_tokens) * p.kv_heads) <= at; ++x) at -= n;
        run_s[0] = x;
        run_s[1] = at;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // The next item for a role: false at the end of the work or after a wait gave up (recorded). One warp.
  int turn = 0;
  auto next_item = [&](Item& w) {
    const int slot = turn & 1;
    const bool ok = __all_sync(0xFFFFFFFFu, wait_own(&item_full[slot], (turn >> 1) & 1, p.err, &until_s));
    if (!ok) return false;
    w = items[slot];
    ++turn;
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[slot]);
    return !w.stop;
  };

  if (warp >= 8) {
    if constexpr (kF32)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    else
      asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 8) {
      // -------------------------------------------------------------- TMA
      const int boxes = kTileKeys / tp.box_rows, b = lane % boxes, panel = lane / boxes;
      const bool mine = lane < boxes * kPanels;
      constexpr int kIn = kF32 ? kStaging : kStages;
      uint64_t *in_full = kF32 ? stage_full : kv_full, *in_empty = kF32 ? stage_empty : kv_empty;
      uint8_t* in = kF32 ? stage : ring;
      Item w;
      bool ok = true;
      int issued = 0, tiles = 0;
      while (ok && next_item(w)) {
        const Plan a = plan_of(w, tp.tokens);
        if (w.count == 0) {
          if (lane == 0) mbar_arrive(&fetch);
          continue;
        }
        if (!kF32 && tiles > 0) ok = wait_own(&q_empty, (tiles - 1) & 1, p.err, &until_s);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        ++tiles;
        if (!kF32 && lane == 0) {  // (F32 queries: the softmax warps)
          const int live = a.n[1] > 0 ? 2 : 1;
          mbar_arrive_expect_tx(&q_full, static_cast<uint32_t>(live * kPanels * tp.tokens * p.group) * 128u);
          for (int i = 0; i < live; ++i)
            for (int h = 0; h < kPanels; ++h)
              tma_load_3d(q_s + (i * kPanels + h) * kPanel, &map_q, 64 * h, w.kvh * p.group,
                          w.c.begin + w.token0 + i * tp.tokens, &q_full);
        }
        // first row of this lane's box in the tensor; outside of it (zero fill) behind the last position
        auto row_of = [&](int tile) -> int32_t {
          const int pos = tile * kTileKeys + b * tp.box_rows;
          if (!mine || tile >= w.first + w.count) return 0;
          if (!p.kv_len) return w.c.begin + pos;
          const int64_t row = pos < a.see_all ? key_row(p, w.c, pos) : -1;
          return static_cast<int32_t>(row >= 0 ? row : p.n_pages * p.page_size);
        };
        int32_t row = row_of(w.first);
        for (int j = 0; j < w.count && ok; ++j) {
          const int32_t next = row_of(w.first + j + 1);
          if (lane == 0) move_on(&until_s);
          if (j == max(0, w.count - 2) && lane == 0) mbar_arrive(&fetch);  // time to look for the next item
          for (int kv = 0; kv < 2 && ok; ++kv) {
            const int st = issued % kIn;
            if (issued >= kIn) ok = wait_own(&in_empty[st], ((issued / kIn) - 1) & 1, p.err, &until_s);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(&in_full[st], kTileBytes);
            __syncwarp();
            if (mine)
              tma_load_3d(in + st * kTileBytes + panel * kPanel + b * tp.box_rows * 128, kv ? &map_v : &map_k,
                          (128 / static_cast<int>(sizeof(T))) * panel, w.kvh, row, &in_full[st]);
            ++issued;
          }
          row = next;
        }
      }
      // the copies in flight land before the shared memory is given back (all have, unless a wait gave up)
      if (!kF32 && tiles > 0) wait_own(&q_full, (tiles - 1) & 1, p.err, &until_s);
      for (int i = max(0, issued - kIn); i < issued; ++i) wait_own(&in_full[i % kIn], (i / kIn) & 1, p.err, &until_s);
    } else if (warp == 9 || (kApart && warp == 11)) {
      // -------------------------------------------------------------- MMA
      // Where P lies apart, each row tile has a warp of its own (9 and 11): a softmax that is ready is never
      // behind the other's. Where P lies in S, one warp serves both in turn, which keeps the row tiles half
      // a step apart: at head size 128 the products are the bound, and both at once would leave the tensor
      // cores idle during both softmaxes. Each whole warp walks this code, so that addresses and
      // descriptors stay warp-uniform (in uniform registers); one elected thread issues. All 512 columns
      // are this CTA's: TMEM addresses start at 0.
      constexpr uint32_t id_s = idesc_of<E>(kTileKeys, false), id_o = idesc_of<E>(kWideO, true);
      constexpr uint32_t id_half = idesc_of<E>(64, true);
      constexpr int kMine = kApart ? 1 : 2;  // row tiles of this warp: from `mine` on
      const int mine = kApart && warp == 11 ? 1 : 0;
      const uint32_t one = elect_one();
      const uint32_t ring_addr = base + 2 * kTileBytes;
      auto scores = [&](int i, int item) {
        const uint64_t dq = smem_desc_sw128(base + i * kTileBytes);
        const uint64_t dk = smem_desc_sw128(ring_addr + (item % kStages) * kTileBytes);
        if constexpr (kF32) {  // hi lo and lo hi first: the accumulator cuts off digits at each step, of small sums less
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            if (ks == 0)
              mma_ss<false>(one, 128 * i, dq, dk + (kPanel >> 4), id_s);
            else
              mma_ss<true>(one, 128 * i, dq + 2 * ks, dk + (kPanel >> 4) + 2 * ks, id_s);
            mma_ss<true>(one, 128 * i, dq + (kPanel >> 4) + 2 * ks, dk + 2 * ks, id_s);
          }
        }
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint64_t adv = (ks / 4) * (kPanel >> 4) + (ks % 4) * 2;
          if (ks == 0 && !kF32)
            mma_ss<false>(one, 128 * i, dq + adv, dk + adv, id_s);
          else
            mma_ss<true>(one, 128 * i, dq + adv, dk + adv, id_s);
        }
        commit_if(one, &s_full[i]);
      };
      auto values = [&](int i, int item, uint32_t add) {
        const uint64_t dv = desc_values(ring_addr + (item % kStages) * kTileBytes);
        const uint32_t o = kColO + kWideO * i, pp = kColP + kStepP * i;
        // F32: P hi times [V hi | V lo], then P lo times V hi onto the columns of the small products; of every 32
        // keys P hi lies in 16 columns and P lo in the next 16
        const auto col = [&](int ks) { return pp + (kF32 ? (ks / 2) * 32 + (ks % 2) * 8 : 8 * ks); };
        mma_ts(one, o, pp, dv, id_o, kF32 ? 0u : add);
#pragma unroll
        for (int ks = 1; ks < kTileKeys / 16; ++ks) mma_ts(one, o, col(ks), dv + ks * (2048 >> 4), id_o, 1u);
        if constexpr (kF32) {
#pragma unroll
          for (int ks = 0; ks < kTileKeys / 16; ++ks) mma_ts(one, o + 64, col(ks) + 16, dv + ks * (2048 >> 4), id_half, 1u);
        }
        commit_if(one, &pv_done[i]);
      };
      // The tile has landed. (A stage is given back only after that, also by a row tile that has no use for it:
      // the other one's use of the stage before is over then.)
      auto landed = [&](int item) { return wait_own(&kv_full[item % kStages], (item / kStages) & 1, p.err, &until_s); };
      Item w;
      bool ok = true;
      int ring_at = 0, tiles = 0;     // ring items and items with keys before this one
      int step[kMine] = {};           // key tiles of each row tile before this item
      while (ok && next_item(w)) {
        const Plan a = plan_of(w, tp.tokens);
        if (w.count == 0) continue;
        int n[kMine];
#pragma unroll
        for (int x = 0; x < kMine; ++x) n[x] = kApart && mine == 1 ? a.n[1] : a.n[x];
        ok = wait_own(&q_full, tiles & 1, p.err, &until_s) && landed(ring_at);
        ++tiles;
#pragma unroll
        for (int x = 0; x < kMine; ++x) {
          if (n[x] == 0) continue;
          // S of the item before has been read (where P lies in S, its value product precedes these MMAs)
          if (kApart && step[x] > 0) ok = ok && wait_own(&s_free[mine + x], (step[x] - 1) & 1, p.err, &until_s);
          if (!ok) continue;
          tc_fence_after();
          scores(mine + x, ring_at);
        }
        if (!ok) break;
        commit_if(one, &kv_empty[ring_at % kStages]);
        if (w.count == 1) commit_if(one, &q_empty);
        for (int j = 0; j < w.count && ok; ++j) {
          const int vi = ring_at + 2 * j + 1, ki = vi + 1;
          const bool more = j + 1 < w.count;
          if (kApart && more) {
            ok = landed(ki);
            if (j + 1 < n[0]) {
              ok = ok && wait_own(&s_free[mine], (step[0] + j) & 1, p.err, &until_s);
              if (!ok) break;
              tc_fence_after();
              scores(mine, ki);
            }
            commit_if(one, &kv_empty[ki % kStages]);
            if (j + 2 == w.count) commit_if(one, &q_empty);
          }
          ok = ok && landed(vi);
          if (!kApart && more) ok = ok && landed(ki);
#pragma unroll
          for (int x = 0; x < kMine; ++x) {
            if (j >= n[x]) continue;
            ok = ok && wait_own(&p_ready[mine + x], (step[x] + j) & 1, p.err, &until_s);
            if (!ok) continue;
            tc_fence_after();
            values(mine + x, vi, j > 0);
            if (!kApart && j + 1 < n[x]) scores(x, ki);
          }
          if (!ok) break;
          commit_if(one, &kv_empty[vi % kStages]);
          if (!kApart && more) {
            commit_if(one, &kv_empty[ki % kStages]);
            if (j + 2 == w.count) commit_if(one, &q_empty);
          }
        }
        ring_at += 2 * w.count;
#pragma unroll
        for (int x = 0; x < kMine; ++x) step[x] += n[x];
      }
      commit_if(one, &drained[mine]);  // no MMA runs on when the TMEM is given back, also after a wait gave up
      __syncwarp();
      mbar_drain(&drained[mine], 0, p.err);
    } else if (kF32 && warp >= 12) {
      // -------------------------------------------------------------- converters
      // An FP32 tile (128 rows of 64 dims, two swizzled panels) becomes the hi and lo panels of an operand tile. Keys: a
      // thread per row, scaled by a power of two after the tile's largest magnitude. Values: 16 rows of four dims a
      // thread, scaled after the largest of each dim. Rows behind the last position become zeros, whatever lies there.
      const int r_ = tid - 384;
      Item w;
      bool ok = true;
      int at = 0, tiles = 0, part = 0;
      while (ok && next_item(w)) {
        const Plan a = plan_of(w, tp.tokens);
        uint32_t most = 0, least = 0xFFFFFFFFu;  // exponents of dims 4 quad .. so far (threads 0-15)
        for (int x = 0; x < 2 * w.count && ok; ++x, ++at) {
          // (opaque, so that the addresses below are not kept in registers across tiles, which spills)
          int r = r_;
          asm volatile("" : "+r"(r));
          const int quad = r & 15, row0 = (r >> 4) * 16;
          const int st = at % kStaging, op = at % kStages, keys = a.see_all - (w.first + (x >> 1)) * kTileKeys;
          ok = wait_own(&stage_full[st], (at / kStaging) & 1, p.err, &until_s);
          if (ok && at >= kStages) ok = wait_own(&kv_empty[op], ((at / kStages) - 1) & 1, p.err, &until_s);
          uint8_t *src = stage + st * kTileBytes, *dst = ring + op * kTileBytes;
          auto chunk = [&](int row, int c) {
            return *reinterpret_cast<const float4*>(src + row * 128 + (c >> 3) * kPanel + (((c & 7) ^ (row & 7)) << 4));
          };
          if (x & 1) {
            if (ok && r >= keys) {  // (in order by the barrier before these rows are read)
#pragma unroll 1
              for (int c = 0; c < 16; ++c)
                *reinterpret_cast<uint4*>(src + r * 128 + (c >> 3) * kPanel + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
            }
            float4 hi = make_float4(0, 0, 0, 0), lo = make_float4(INFINITY, INFINITY, INFINITY, INFINITY);
            const auto range = [&](const float4& v, const float4& u) {
              hi = make_float4(max3_abs(hi.x, v.x, u.x), max3_abs(hi.y, v.y, u.y), max3_abs(hi.z, v.z, u.z), max3_abs(hi.w, v.w, u.w));
              lo = make_float4(min3_abs(lo.x, v.x, u.x), min3_abs(lo.y, v.y, u.y), min3_abs(lo.z, v.z, u.z), min3_abs(lo.w, v.w, u.w));
            };
            if (keys >= kTileKeys) {
#pragma unroll
              for (int k = 0; k < 16; k += 2) range(chunk(row0 + k, quad), chunk(row0 + k + 1, quad));
            } else {  // the last valid row in place of those behind it
#pragma unroll 8
              for (int k = 0; k < 16; k += 2)
                range(chunk(min(row0 + k, keys - 1), quad), chunk(min(row0 + k + 1, keys - 1), quad));
            }
            if (lo.x == 0.f || lo.y == 0.f || lo.z == 0.f || lo.w == 0.f) {  // the least but zero
              lo = make_float4(INFINITY, INFINITY, INFINITY, INFINITY);
              const auto some = [](float l, float v) { return v != 0.f ? min3_abs(l, v, v) : l; };
              if (hi.x != 0.f || hi.y != 0.f || hi.z != 0.f || hi.w != 0.f) {
#pragma unroll 1
                for (int k = 0; k < 16; ++k) {
                  const float4 v = chunk(min(row0 + k, keys - 1), quad);
                  lo = make_float4(some(lo.x, v.x), some(lo.y, v.y), some(lo.z, v.z), some(lo.w, v.w));
                }
              }
            }
            // biased exponents, 0 for zeros alone; of a dim of zeros the least is 255
            const auto exponent = [](float v) { return max(__float_as_uint(v) >> 23, min(__float_as_uint(v), 1u)); };
            uint32_t high = exponent(hi.x) | exponent(hi.y) << 8 | exponent(hi.z) << 16 | exponent(hi.w) << 24;
            uint32_t low = exponent(lo.x) | exponent(lo.y) << 8 | exponent(lo.z) << 16 | exponent(lo.w) << 24;
            high = __vmaxu4(high, __shfl_xor_sync(0xFFFFFFFFu, high, 16));
            low = __vminu4(low, __shfl_xor_sync(0xFFFFFFFFu, low, 16));
            if (lane < 16) {
              reinterpret_cast<uint32_t*>(&dims_s[0][quad])[warp - 12] = high;
              reinterpret_cast<uint32_t*>(&dims_s[1][quad])[warp - 12] = low;
            }
            ok = all_converters(ok);  // also orders dims_s
            if (!ok) break;
            const uint4 h = dims_s[0][quad];
            high = __vmaxu4(__vmaxu4(h.x, h.y), __vmaxu4(h.z, h.w));
            // (a dim with an infinity makes NaN of its sums: its scale only has to be a number)
            const auto of = [](uint32_t high, int y) { return max(-100, min(127, static_cast<int>(high >> (8 * y) & 255u) - 127)); };
            const float4 scale = make_float4(power_of_two(kTop - of(high, 0)), power_of_two(kTop - of(high, 1)),
                                             power_of_two(kTop - of(high, 2)), power_of_two(kTop - of(high, 3)));
            if (r < 16) {
              // (a unit times its scale is 2^-kRaise)
              const auto unit = [](float s) { return __uint_as_float(((254u - kRaise) << 23) - __float_as_uint(s)); };
              unit_s[part][quad] = make_float4(unit(scale.x), unit(scale.y), unit(scale.z), unit(scale.w));
              const uint4 l = dims_s[1][quad];
              most = __vmaxu4(most, high);
              least = __vminu4(least, __vminu4(__vminu4(l.x, l.y), __vminu4(l.z, l.w)));
              uint32_t wide = 0;
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const int bound = of(most, y) - kTop - kRaise + 127;  // the largest unit
                if (static_cast<int>(least >> (8 * y) & 255u) < bound) wide |= static_cast<uint32_t>(bound) << (8 * y);
              }
              reinterpret_cast<uint32_t*>(wide_s[tiles & 1])[quad] = wide;
            }
            part = part == 2 ? 0 : part + 1;
#pragma unroll 1
            for (int k0 = 0; k0 < 16; k0 += 8) {
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                uint2 a, b;
                split4<true>(chunk(row0 + k0 + k, quad), scale, a, b);
                uint8_t* to = dst + (row0 + k0 + k) * 128 + (((quad >> 1) ^ k) << 4) + (quad & 1) * 8;
                *reinterpret_cast<uint2*>(to) = a;
                *reinterpret_cast<uint2*>(to + kPanel) = b;
              }
            }
            __syncwarp();  // unit_s and wide_s, before exp_full
          } else {
            const bool valid = r < keys;
            float m = 0.f;
            if (valid) {
              float4 hi = make_float4(0, 0, 0, 0);
#pragma unroll
              for (int c = 0; c < 16; c += 2) {
                const float4 v = chunk(r, c), u = chunk(r, c + 1);
                hi = make_float4(max3_abs(hi.x, v.x, u.x), max3_abs(hi.y, v.y, u.y), max3_abs(hi.z, v.z, u.z), max3_abs(hi.w, v.w, u.w));
              }
              m = fmaxf(fmaxf(hi.x, hi.y), fmaxf(hi.z, hi.w));
              if (!(m <= 3.402823466e38f)) {  // an infinity
                m = 0.f;
#pragma unroll 1
                for (int c = 0; c < 16; ++c) m = finite_max(m, chunk(r, c));
              }
            }
            const uint32_t bits = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(m));
            float* ms = max_s[(at >> 1) & 1];
            if (lane == 0) ms[warp - 12] = __uint_as_float(bits);
            ok = all_converters(ok);  // also orders max_s
            if (!ok) break;
            const int e = exponent_of(fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3])));
            const float f = power_of_two(kTop - e);
            const float4 scale = make_float4(f, f, f, f);
            if (r == 0) exp_s[at & 7] = e;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              uint2 a[2] = {}, b[2] = {};
              if (valid) {
                split4<false>(chunk(r, 2 * c), scale, a[0], b[0]);
                split4<false>(chunk(r, 2 * c + 1), scale, a[1], b[1]);
              }
              *reinterpret_cast<uint4*>(dst + r * 128 + ((c ^ (r & 7)) << 4)) = make_uint4(a[0].x, a[0].y, a[1].x, a[1].y);
              *reinterpret_cast<uint4*>(dst + r * 128 + kPanel + ((c ^ (r & 7)) << 4)) = make_uint4(b[0].x, b[0].y, b[1].x, b[1].y);
            }
          }
          if (r == 0) mbar_arrive(&exp_full[at & 7]);
          fence_proxy_async();
          mbar_arrive(&kv_full[op]);
          mbar_arrive(&stage_empty[st]);
        }
        tiles += w.count > 0;
      }
    } else if (warp == 10) {
      // -------------------------------------------------------------- scheduler
      // Items are numbered key head by key head, the pairs of row tiles of a sequence last to first (the last see
      // the most keys). A CTA begins with the item of its own number; when its loads are nearly issued it
      // takes over the next CTA that the hardware has not started, so the GPU stays balanced whatever the
      // items take. Sequences are counted 32 at a time.
      // With a workspace (few items for the GPU, or ragged ones) the line of all key tiles is cut into equal runs
      // instead, one per CTA, and items are cut where the runs end.
      const int total = tp.tiles * p.kv_heads, pair_tokens = 2 * tp.tokens;
      int sent = 0;
      bool ok = true;
      auto send = [&](const Item& w) {
        const int slot = sent & 1;
        if (sent >= 2) ok = wait_own(&item_empty[slot], ((sent >> 1) - 1) & 1, p.err, &until_s);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) return;
        if (lane == 0) {
          items[slot] = w;
          mbar_arrive(&item_full[slot]);
        }
        __syncwarp();
        ++sent;
      };
      Item w;
      w.stop = 0;
      if constexpr (kRuns) {
        const int line = run_s[2], n_runs = run_s[3];
        if (line > 0 && static_cast<int>(blockIdx.x) < n_runs) {
          const Runs runs(line, n_runs);
          const int end = static_cast<int>(runs.begin(blockIdx.x + 1));
          int seq = run_s[0], at = run_s[1], left = end - static_cast<int>(runs.begin(blockIdx.x)), parts = 0;
          while (left > 0 && ok && seq < p.n_seqs) {
            const int weight = weight_of(p, seq, pair_tokens);  // 0: nothing to do there
            if (at >= weight * p.kv_heads) {
              ++seq;
              at = 0;
              continue;
            }
            chunk_of_seq(p, seq, w.c);
            w.kvh = at / weight;
            int off = at - w.kvh * weight, tiles = 0;
            for (w.token0 = 0;; w.token0 += pair_tokens) {  // the pair that holds the place
              tiles = tiles_of_pair(w.c, w.token0, pair_tokens);
              if (off < kItemCost + tiles) break;
              off -= kItemCost + tiles;
            }
            const int step = min(kItemCost + tiles - off, left), to = off + step - kItemCost;
            left -= step;
            at += step;
            // (a run that ends before the item's first key tile leaves it to the next; rows that see nothing
            // belong to the run that holds the end of their item)
            if (to <= 0 && !(tiles == 0 && to == 0)) continue;
            w.first = max(0, off - kItemCost);
            w.count = to - w.first;
            const bool whole = w.count == tiles;
            w.slot = whole ? -1 : min(parts, 1);
            ++parts;
            if (!whole && w.first == 0 && lane == 0)  // its last piece is in the run that holds its end
              tp.joins[blockIdx.x] = TcJoin{w.c, w.kvh, w.token0, w.slot,
                                            static_cast<int>(runs.at(end - 1 + (tiles - to))) - static_cast<int>(blockIdx.x) + 1};
            send(w);
          }
        }
      } else {
        int asks = 0, s0 = 0, before = 0, last_tile = 0;  // the scan stands at sequence s0 with `before` tiles before it
        // the number of the next item, -1 behind the last
        auto next_number = [&]() -> int {
          if (lane == 0) {
            mbar_arrive_expect_tx(&asked, 16);
            ask_next_cta(&answer, &asked);
          }
          __syncwarp();
          ok = __all_sync(0xFFFFFFFFu, wait_own(&asked, asks & 1, p.err, &until_s));
          ++asks;
          if (!ok) return -1;
          const int x = next_cta(&answer);
          fence_proxy_async();  // the answer has been read before the next one may be written
          __syncwarp();
          return x;
        };
        for (int wi = static_cast<int>(blockIdx.x); wi >= 0 && ok; wi = next_number()) {
          const int kvh = wi / tp.tiles, tile = wi - kvh * tp.tiles;
          if (wi >= total) continue;
          int64_t seq = -1, index = 0;
          if (tp.tiles_per_seq > 0) {
            seq = tile / tp.tiles_per_seq;
            index = tp.tiles_per_seq - 1 - (tile - seq * tp.tiles_per_seq);
          } else {
            if (tile < last_tile) s0 = before = 0;  // another key head
            last_tile = tile;
            for (; s0 < p.n_seqs; s0 += 32) {
              int64_t m = s0 + lane < p.n_seqs ? static_cast<int64_t>(p.cu[s0 + lane + 1]) - p.cu[s0 + lane] : 0;
              // lengths that make no sense get one tile, which records them
              const int n = m < 0 || m > p.n_rows ? 1 : static_cast<int>((m + pair_tokens - 1) / pair_tokens);
              int inc = n;
#pragma unroll
              for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xFFFFFFFFu, inc, o);
                if (lane >= o) inc += up;
              }
              const uint32_t hit = __ballot_sync(0xFFFFFFFFu, tile >= before + inc - n && tile < before + inc);
              if (hit) {
                const int l = __ffs(hit) - 1;
                seq = s0 + l;
                index = __shfl_sync(0xFFFFFFFFu, before + inc - 1 - tile, l);
                break;
              }
              before += __shfl_sync(0xFFFFFFFFu, inc, 31);
            }
          }
          if (seq < 0 || !chunk_of_seq(p, seq, w.c) || index * pair_tokens >= w.c.end - w.c.begin) continue;
          w.kvh = kvh;
          w.token0 = static_cast<int>(index) * pair_tokens;
          w.first = 0;
          w.count = tiles_of_pair(w.c, w.token0, pair_tokens);
          w.slot = -1;
          send(w);
          if (ok) ok = __all_sync(0xFFFFFFFFu, wait_own(&fetch, (sent - 1) & 1, p.err, &until_s));
        }
      }
      if (ok) {
        w.stop = 1;
        send(w);
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    if constexpr (kF32)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
    else
      asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int i = warp >> 2, r = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t s_addr = tmem + lanes + 128 * i, o_addr = tmem + lanes + kColO + kWideO * i;
    const uint32_t p_addr = tmem + lanes + kColP + kStepP * i;
    const int token = r / p.group;  // of the row tile
    const float scale2 = p.scale * 1.4426950408889634f;
    bool ok = true;
    int ring_at = 0, step = 0;  // ring items, and key tiles of this row tile, before this item
    int tiles = 0;              // items with keys before this one
    for (;; ++turn) {
      const int slot = turn & 1;
      // (read again where needed: the registers are for S)
      ok = ok && __all_sync(0xFFFFFFFFu, wait_own(&item_full[slot], (turn >> 1) & 1, p.err, &until_s));
      if (!ok || items[slot].stop) break;
      int n, first, count, see_all, sees, see_first;
      {
        const Item w = items[slot];
        const Plan a = plan_of(w, tp.tokens);
        n = a.n[i];
        first = w.first;
        count = w.count;
        see_all = a.see_all;
        const int row0 = w.c.begin + w.token0 + i * tp.tokens;
        sees = token < a.tok[i] ? seen_by(w.c, row0 + token) : 0;
        see_first = a.tok[i] ? seen_by(w.c, row0) : 0;
      }
      uint64_t total[2] = {0, 0};  // pairs of FP32 zeros
      float ref = 0.f;
      int exp_q = 0;                // F32: exponent of this row's query
      uint64_t acc[kF32 ? D / 2 : 1] = {};  // F32: O of the key tiles before, pairs
      if (kF32 && count > 0) {
        // this row's query, scaled by a power of two, as the hi and lo rows of the Q operand
        if (tiles > 0) ok = ok && wait_own(&q_empty, (tiles - 1) & 1, p.err, &until_s);
        const int64_t row = items[slot].c.begin + items[slot].token0 + i * tp.tokens + token;
        const int head = items[slot].kvh * p.group + r - token * p.group;
        const bool live = token < plan_of(items[slot], tp.tokens).tok[i];
        const float* q = static_cast<const float*>(p.q) + row * p.q_stride + static_cast<int64_t>(head) * p.head_dim;
        float4 v[16];
        float m = 0.f;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          v[c] = live && 4 * c < p.head_dim ? *reinterpret_cast<const float4*>(q + 4 * c) : make_float4(0, 0, 0, 0);
          m = finite_max(m, v[c]);
        }
        exp_q = exponent_of(m);
        uint8_t* dst = q_s + i * kTileBytes + r * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float f = power_of_two(kTop - exp_q);
          const float4 scale = make_float4(f, f, f, f);
          uint2 hi[2], lo[2];
          split4<false>(v[2 * c], scale, hi[0], lo[0]);
          split4<false>(v[2 * c + 1], scale, hi[1], lo[1]);
          *reinterpret_cast<uint4*>(dst + ((c ^ (r & 7)) << 4)) = make_uint4(hi[0].x, hi[0].y, hi[1].x, hi[1].y);
          *reinterpret_cast<uint4*>(dst + kPanel + ((c ^ (r & 7)) << 4)) = make_uint4(lo[0].x, lo[0].y, lo[1].x, lo[1].y);
        }
        fence_proxy_async();
        mbar_arrive(&q_full);
      }
      tiles += count > 0;
      bool coarse = false;  // F32: a row that is computed again
      if constexpr (kF32) {
        // O of one key tile at a time is added up here, in registers: the tensor cores' accumulators cut off instead
        // of rounding, which over a long row would shrink it (by 5e-6 at 8192 keys). S is read 32 columns at a time
        // to leave room for that.
        int high_k = -126;
        const auto take = [&](int j, float back) {  // O of key tile j
          const float4* units = unit_s[(ring_at / 2 + j) % 3];
          const uint64_t backs = pair(back, back);
#pragma unroll
          for (int q = 0; q < D / 32; ++q) {
            uint32_t o[32];
            load_o<true>(o_addr + 32 * q, o);
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 u = units[8 * q + e / 4];
              uint64_t* a = acc + 16 * q + e / 2;
              a[0] = fma2(fma2(pair(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), pair(u.x, u.y), a[0]), backs, 0);
              a[1] = fma2(fma2(pair(__uint_as_float(o[e + 2]), __uint_as_float(o[e + 3])), pair(u.z, u.w), a[1]), backs, 0);
            }
          }
        };
        for (int j = 0; j < n; ++j, ++step) {
          ok = ok && wait_own(&s_full[i], step & 1, p.err, &until_s);
          if (!__all_sync(0xFFFFFFFFu, ok)) break;
          tc_fence_after();
          const int key0 = (first + j) * kTileKeys;
          const bool edge = key0 + kTileKeys > see_first;
          const int limit = sees - key0;
          // groups of 32 columns that some row of the warp sees
          const int groups = edge ? min(4, (max(0, __reduce_max_sync(0xFFFFFFFFu, limit)) + 31) / 32) : 4;
          uint32_t s[32];
          const auto load = [&](int q) {  // columns 32 q ..
            tmem_ld32(s_addr + 32 * q, s);
            tmem_wait_ld();
            after_wait(s);
            if (edge) {
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (k + 32 * q >= limit) s[k] = 0xFF800000u;  // -inf
            }
          };
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
          for (int q = 0; q < groups; ++q) {
            load(q);
#pragma unroll
            for (int k = 0; k < 32; k += 8)
#pragma unroll
              for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(s[k + e]), __uint_as_float(s[k + e + 4]));
          }
          const int ki = ring_at + 2 * j;
          ok = wait_own(&exp_full[ki & 7], (ki >> 3) & 1, p.err, &until_s);
          high_k = max(high_k, exp_s[ki & 7]);
          const float factor = scale2 * power_of_two(max(-120, min(120, exp_q + exp_s[ki & 7] - 2 * kTop)));
          const float high = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * factor;
          if (j == 0) {
            ref = high == -INFINITY ? 0.f : high;
          } else {
            const bool move = high - ref > kLazy<T>;
            const float back = move ? ex2(ref - high) : 1.f;
            if (move) ref = high;
            total[0] = fma2(total[0], pair(back, back), 0);
            total[1] = fma2(total[1], pair(back, back), 0);
            ok = ok && wait_own(&pv_done[i], (step - 1) & 1, p.err, &until_s) &&
                 wait_own(&exp_full[(ki - 1) & 7], ((ki - 1) >> 3) & 1, p.err, &until_s);  // (its units; long there)
            if (!__all_sync(0xFFFFFFFFu, ok)) break;
            tc_fence_after();
            take(j - 1, back);
          }
          const uint64_t scale_pair = pair(factor, factor), nref = pair(-ref, -ref);
#pragma unroll 1
          for (int q = 0; q < 4; ++q) {  // (P takes the place of the columns of S that have been read)
            uint32_t hi[16] = {}, lo[16] = {};
            if (q < groups) {
              load(q);
              weights32_split(s, scale_pair, nref, total, hi, lo);
            }
            tmem_st16(p_addr + 32 * q, hi);
            tmem_st16(p_addr + 32 * q + 16, lo);
          }
          if (!__all_sync(0xFFFFFFFFu, ok)) break;
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&p_ready[i]);
        }
        if (n > 0) {
          const int own = ring_at + 2 * n - 1, last = ring_at + 2 * count - 1;  // the item's last value tile: wide_s stands
          ok = ok && wait_own(&pv_done[i], (step - 1) & 1, p.err, &until_s) && wait_own(&exp_full[own & 7], (own >> 3) & 1, p.err, &until_s);
          ok = __all_sync(0xFFFFFFFFu, ok);
          tc_fence_after();
          take(n - 1, 1.f);
          ok = ok && wait_own(&exp_full[last & 7], (last >> 3) & 1, p.err, &until_s);
          ok = __all_sync(0xFFFFFFFFu, ok);
        }
        coarse = p.scale * power_of_two(max(-126, min(127, exp_q + high_k))) > kScoreRange;
        if (n > 0 && sees > 0) {
          const uint4* wide = wide_s[(tiles - 1) & 1];
          const uint4 a = wide[0], b = wide[1], c = wide[2], d = wide[3];
          if ((a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w | c.x | c.y | c.z | c.w | d.x | d.y | d.z | d.w) != 0) {
            float ta, tb;
            unpair(add2(total[0], total[1]), ta, tb);
            const float sum = (ta + tb) * power_of_two(-kRaise);
            const auto far = [&](uint32_t four, const uint64_t* acc) {
              float x[4];
              unpair(acc[0], x[0], x[1]);
              unpair(acc[1], x[2], x[3]);
#pragma unroll
              for (int y = 0; y < 4; ++y)  // (a bound of 0 holds for none)
                coarse = coarse || fabsf(x[y]) < sum * __uint_as_float((four >> (8 * y) & 255u) << 23);
            };
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint4 w = e == 0 ? a : e == 1 ? b : e == 2 ? c : d;
              far(w.x, acc + 8 * e), far(w.y, acc + 8 * e + 2), far(w.z, acc + 8 * e + 4), far(w.w, acc + 8 * e + 6);
            }
          }
        }
      } else {
        for (int j = 0; j < n; ++j, ++step) {
          ok = wait_own(&s_full[i], step & 1, p.err, &until_s);
          if (!__all_sync(0xFFFFFFFFu, ok)) break;
          tc_fence_after();
          uint32_t s[128];
          const int key0 = (first + j) * kTileKeys;
          const bool edge = key0 + kTileKeys > see_first;
          const int limit = sees - key0;
#pragma unroll
          for (int q = 0; q < 4; ++q) tmem_ld32(s_addr + 32 * q, s + 32 * q);
          tmem_wait_ld();
#pragma unroll
          for (int q = 0; q < 4; ++q) after_wait(s + 32 * q);
          if (kApart) {
            tc_fence_before();
            mbar_arrive(&s_free[i]);
          }
          if (edge) {
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
          const uint64_t scale_pair = pair(scale2, scale2);
          const float high = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
          // P and O of the key tile before are free once its value product is done
          const auto before_done = [&] {
            if (j > 0) ok = ok && wait_own(&pv_done[i], (step - 1) & 1, p.err, &until_s);
            tc_fence_after();
          };
          if (j == 0) {
            ref = high == -INFINITY ? 0.f : high;
          } else {
            const bool move = high - ref > kLazy<T>;
            if (__any_sync(0xFFFFFFFFu, move)) {
              before_done();
              const float back = move ? ex2(ref - high) : 1.f;
              if (move) ref = high;
              total[0] = fma2(total[0], pair(back, back), 0);
              total[1] = fma2(total[1], pair(back, back), 0);
#pragma unroll 1
              for (int q = 0; q < static_cast<int>(kWideO) / 32; ++q) {
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
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t x[16];
            weights32<T>(s + 32 * q, scale_pair, nref, total, x);
            if (q == 0) before_done();
            tmem_st16(p_addr + 16 * q, x);
          }
          if (!__all_sync(0xFFFFFFFFu, ok)) break;
          if (key0 + kTileKeys > see_all) {
            // values behind the last position: whatever lies there would meet weights of zero, and 0 times
            // infinity is NaN, so it becomes zero
            const int item = ring_at + 2 * j + 1, st = item % kStages;
            ok = wait_own(&kv_full[st], (item / kStages) & 1, p.err, &until_s);
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
      }
      ring_at += 2 * count;
      float ta, tb;
      unpair(add2(total[0], total[1]), ta, tb);
      const float row_sum = kF32 ? (ta + tb) * power_of_two(-kRaise) : ta + tb;
      if (!kF32 && ok && n > 0) ok = wait_own(&pv_done[i], (step - 1) & 1, p.err, &until_s);
      tc_fence_after();
      ok = __all_sync(0xFFFFFFFFu, ok);
      const Item w = items[slot];
      const Plan a = plan_of(w, tp.tokens);
      const int row0 = w.c.begin + w.token0 + i * tp.tokens;
      const bool live = token < a.tok[i];

      if (!kRuns || w.slot < 0) {
        const float inv = sees > 0 && row_sum != 0.f ? 1.f / row_sum : 0.f;
        const int64_t row = row0 + token;
        const int head = w.kvh * p.group + r - token * p.group;
        T* out = static_cast<T*>(p.out) + (row * p.heads + head) * p.head_dim;
        bool finite = true;
        if constexpr (kF32) {
          if (live && ok) {
#pragma unroll
            for (int e = 0; e < D; e += 4) {
              float v[4];
              unpair(fma2(acc[e / 2], pair(inv, inv), 0), v[0], v[1]);
              unpair(fma2(acc[e / 2 + 1], pair(inv, inv), 0), v[2], v[3]);
#pragma unroll
              for (int y = 0; y < 4; ++y) finite = finite && fabsf(v[y]) <= 3.402823466e38f;
              if (e < p.head_dim) *reinterpret_cast<float4*>(out + e) = make_float4(v[0], v[1], v[2], v[3]);
            }
          }
        } else {
#pragma unroll 1
          for (int q = 0; q < D / 32; ++q) {
            uint32_t o[32];
            if (n > 0) load_o<false>(o_addr + 32 * q, o);
            if (live && ok) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                uint32_t x[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  const float u = inv == 0.f ? 0.f : __uint_as_float(o[e + 2 * y]) * inv;
                  const float v = inv == 0.f ? 0.f : __uint_as_float(o[e + 2 * y + 1]) * inv;
                  finite = finite && fabsf(u) <= 3.402823466e38f && fabsf(v) <= 3.402823466e38f;
                  x[y] = pack2<T>(u, v);
                }
                if (32 * q + e < p.head_dim)
                  *reinterpret_cast<uint4*>(out + 32 * q + e) = make_uint4(x[0], x[1], x[2], x[3]);
              }
            }
          }
        }
        // a row may not be reached by what lies at positions it does not see
        const uint32_t again = __ballot_sync(0xFFFFFFFFu, live && ok && coarse && sees > 0);
        uint32_t redo = again | __ballot_sync(0xFFFFFFFFu, live && ok && !finite && sees < see_all);
        while (redo) {
          const int l = __ffs(redo) - 1;
          redo &= redo - 1;
          const int64_t row_l = __shfl_sync(0xFFFFFFFFu, row, l);
          const int head_l = __shfl_sync(0xFFFFFFFFu, head, l);
          if ((again >> l & 1) || reached_from_behind<T>(p, w.c, row_l, w.kvh, see_all))
            attend_row<T>(p, w.c, row_l, head_l, &until_s);
        }
      } else {
        // a piece: row `tid` of the slot; 16-byte pieces of the rows lie side by side, so that a warp's stores do
        float* slot_o = tp.slots + (static_cast<int64_t>(blockIdx.x) * 2 + w.slot) * (256 * (D + 2));
        if (live) {
          // a row that saw none of these keys takes no part; infinity: to be computed again
          slot_o[tid] = row_sum == 0.f ? -INFINITY : coarse ? INFINITY : ref;
          slot_o[256 + tid] = row_sum;
        }
        if constexpr (kF32) {
          if (live) {
#pragma unroll
            for (int e = 0; e < D / 4; ++e) {
              float x[4];
              unpair(acc[2 * e], x[0], x[1]);
              unpair(acc[2 * e + 1], x[2], x[3]);
              *reinterpret_cast<float4*>(slot_o + 512 + (e * 256 + tid) * 4) = make_float4(x[0], x[1], x[2], x[3]);
            }
          }
        } else {
#pragma unroll 1
          for (int q = 0; q < D / 32; ++q) {
            uint32_t o[32];
            if (n > 0) {
              load_o<false>(o_addr + 32 * q, o);
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = 0u;
            }
            if (live) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<uint4*>(slot_o + 512 + ((8 * q + e) * 256 + tid) * 4) =
                    make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
          }
        }
      }
      tc_fence_before();  // O has been read before this warp's next p_ready lets the MMAs write it
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
    }
  }
  tc_fence_before();
  cta_barrier<kThreads>();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

// Joins the pieces of the item that begins at the end of CTA blockIdx.x's run. A block takes 32 of its 256 rows,
// a lane per row; a warp takes every eighth 16 bytes of the rows.
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_tc_join_kernel(const __grid_constant__ TcParams tp) {
  constexpr int kMine = D / 4 / 8;
  __shared__ int redo_s[32];
  const AttnParams& p = tp.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = blockIdx.y * 32 + lane;
  if (threadIdx.x < 32) redo_s[threadIdx.x] = 0;
  pdl_wait();
  const TcJoin j = tp.joins[blockIdx.x];
  if (j.parts <= 1) return;
  __syncthreads();
  constexpr int64_t kSlot = 256 * (D + 2);
  const float* slots = tp.slots + static_cast<int64_t>(blockIdx.x) * 2 * kSlot;
  auto slot = [&](int x) { return slots + (2 * x + (x == 0 ? j.first : 0)) * kSlot; };
  const int i = r >> 7, token = (r & 127) / p.group, head = j.kvh * p.group + (r & 127) - token * p.group;
  const int tok = min(tp.tokens, j.c.end - j.c.begin - j.token0 - i * tp.tokens);
  const bool live = token < tok;
  const int row = j.c.begin + j.token0 + i * tp.tokens + token;
  if (live) {
    float mx = -INFINITY;
#pragma unroll 4
    for (int x = 0; x < j.parts; ++x) mx = fmaxf(mx, slot(x)[r]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float l = 0.f;
    float4 acc[kMine];
#pragma unroll
    for (int k = 0; k < kMine; ++k) acc[k] = make_float4(0, 0, 0, 0);
#pragma unroll 2
    for (int x = 0; x < j.parts; ++x) {
      const float* o = slot(x);
      const float f = ex2(o[r] - ref);
      l += f * o[256 + r];
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(o + 512 + ((warp + 8 * k) * 256 + r) * 4);
        acc[k].x += f * v.x, acc[k].y += f * v.y, acc[k].z += f * v.z, acc[k].w += f * v.w;
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* out = static_cast<T*>(p.out) + (static_cast<int64_t>(row) * p.heads + head) * p.head_dim;
    bool finite = true;
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const float v[4] = {acc[k].x * inv, acc[k].y * inv, acc[k].z * inv, acc[k].w * inv};
#pragma unroll
      for (int e = 0; e < 4; ++e) finite = finite && fabsf(v[e]) <= 3.402823466e38f;
      const int d = 4 * (warp + 8 * k);
      if (d >= p.head_dim) continue;
      if constexpr (is_f32<T>)
        *reinterpret_cast<float4*>(out + d) = make_float4(v[0], v[1], v[2], v[3]);
      else
        *reinterpret_cast<uint2*>(out + d) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    }
    if (mx == INFINITY)
      redo_s[lane] = 2;
    else if (!finite)
      redo_s[lane] = 1;
  }
  __syncthreads();
  const int see_all = keys_of(j.c, min(j.c.end - j.c.begin, j.token0 + 2 * tp.tokens));
  for (int x = warp; x < 32; x += 8) {
    const int rx = __shfl_sync(0xFFFFFFFFu, row, x), hx = __shfl_sync(0xFFFFFFFFu, head, x);
    if (redo_s[x] == 2 ||
        (redo_s[x] && seen_by(j.c, rx) < see_all && reached_from_behind<T>(p, j.c, rx, j.kvh, see_all)))
      attend_row<T>(p, j.c, rx, hx);
  }
}

template <typename T, int D>
int launch(const AttnParams& p, int64_t max_new, int sms, void* work, cudaStream_t s) {
  TcParams tp;
  tp.a = p;
  tp.tokens = kTileRows / p.group;
  const int type = is_f32<T> ? EFG_F32 : std::is_same_v<T, __nv_bfloat16> ? EFG_BF16 : EFG_F16;
  const int64_t kv_rows = p.kv_len ? p.n_pages * p.page_size : p.n_rows;
  tp.box_rows = p.kv_len ? static_cast<int>(std::min<int64_t>(p.page_size, kTileKeys)) : kTileKeys;
  CUtensorMap mq, mk, mv;
  // (F32 queries do not come by TMA: their map is made all the same, it checks the rows)
  if (!encode_heads_map(&mq, type, p.q, p.head_dim, p.heads, p.n_rows, p.q_stride, p.group, tp.tokens) ||
      !encode_heads_map(&mk, type, p.k, p.head_dim, p.kv_heads, kv_rows, p.k_stride, 1, tp.box_rows) ||
      !encode_heads_map(&mv, type, p.v, p.head_dim, p.kv_heads, kv_rows, p.v_stride, 1, tp.box_rows))
    return fail(EFG_ECUDA, "attention: the driver rejects a tensor map");
  const int64_t pair_tokens = 2 * tp.tokens, per_seq = (max_new + pair_tokens - 1) / pair_tokens;
  const int64_t fixed = p.n_seqs * per_seq, bound = p.n_rows / pair_tokens + p.n_seqs;
  const int64_t tiles = std::min(fixed, bound);
  if (tiles * p.kv_heads > 0x3FFFFFFFll) return fail(EFG_EINVAL, "attention: too many rows");
  tp.tiles = static_cast<int>(tiles);
  tp.tiles_per_seq = fixed <= bound ? static_cast<int>(per_seq) : 0;
  const auto fn = work ? attn_tc_kernel<T, D, true> : attn_tc_kernel<T, D, false>;
  if (int st = ensure_smem_attr(reinterpret_cast<const void*>(fn), smem_bytes<T, D>)) return st;
  cudaLaunchConfig_t cf{};
  tp.joins = static_cast<TcJoin*>(work);
  tp.slots = work ? reinterpret_cast<float*>(tp.joins + sms) : nullptr;
  // a CTA per run, or per item; those that run take over the others
  cf.gridDim = dim3(static_cast<unsigned>(work ? sms : tiles * p.kv_heads));
  cf.blockDim = dim3(threads<T>);
  cf.dynamicSmemBytes = smem_bytes<T, D>;
  cf.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cf.attrs = attr;
  cf.numAttrs = 1;
  EFG_TRY_CUDA(cudaLaunchKernelEx(&cf, fn, tp, mq, mk, mv), "attention launch");
  if (!work) return EFG_OK;
  cf.gridDim = dim3(static_cast<unsigned>(sms), 8);
  cf.blockDim = dim3(256);
  cf.dynamicSmemBytes = 0;
  EFG_TRY_CUDA(cudaLaunchKernelEx(&cf, attn_tc_join_kernel<T, D>, tp), "attention launch");
  return EFG_OK;
}

}  // namespace

bool attn_tc_takes(int type, const AttnParams& p) {
  if ((type == EFG_F32 && p.head_dim > 64) || !(p.scale > 0.f) || p.group > kTileRows || reinterpret_cast<uintptr_t>(p.out) % 16) return false;
  if (p.q_stride == 0 || p.k_stride == 0 || p.v_stride == 0) return false;
  if (p.kv_len) {  // whole boxes of a page, whole 8-row groups of the swizzle
    if (p.n_pages == 0 || p.page_size < 8 || (p.page_size & (p.page_size - 1))) return false;
  }
  const int64_t max_new = p.kv_len ? std::min(p.max_new, p.n_rows) : p.n_rows;
  // Prompts above the decode kernel's rows: 9.8 against 13.4 us at 23 BF16 tokens, 14.1 against 18.7 in F32. Over
  // pages, where the warp-level kernel splits the keys over clusters, from 64 rows on (8 sequences of 1000
  // positions and 3 to 8 new tokens: 17.8 against 16.2 us; F32 33 against 29).
  return attn_mma_takes(type, p) && max_new * p.group > (p.kv_len ? 64 : kDecodeRows);
}

size_t attn_tc_workspace(const AttnParams& p, int sms) {
  // Prompts bring no workspace. More than six items a CTA are not cut: where their lengths are alike that saves the
  // pieces' way through memory (130 chunks of 100 tokens over 2000 positions, 8 key heads of 128: 553 us, cut 595; 255
  // single tokens over 1000 positions beside 512 over 4000: 325, cut 352). One long item among short ones is then walked
  // by one CTA a key head (64 tokens over 65536 positions beside 255 single ones over 200: 1090 us, cut 219); the
  // host does not know the lengths. The line's weight is a 32-bit number.
  if (!p.kv_len) return 0;
  const int64_t max_new = std::min(p.max_new, p.n_rows), pair_tokens = 2 * (kTileRows / p.group);
  const int64_t tiles = std::min(p.n_seqs * ((max_new + pair_tokens - 1) / pair_tokens), p.n_rows / pair_tokens + p.n_seqs);
  const int64_t max_keys = p.max_pages * p.page_size;
  if (tiles * p.kv_heads > 6 * sms || tiles * p.kv_heads > 0x7FFFFFFFll / (max_keys / kTileKeys + 1 + kItemCost)) return 0;
  return static_cast<size_t>(sms) * (sizeof(TcJoin) + 2 * 256 * ((p.head_dim <= 64 ? 64 : 128) + 2) * sizeof(float));
}

int launch_attn_tc(int type, const AttnParams& p, int sms, void* work, cudaStream_t s) {
  const int64_t max_new = p.kv_len ? std::min(p.max_new, p.n_rows) : p.n_rows;
  if (type == EFG_F32) return launch<float, 64>(p, max_new, sms, work, s);
  if (type == EFG_F16)
    return p.head_dim <= 64 ? launch<__half, 64>(p, max_new, sms, work, s) : launch<__half, 128>(p, max_new, sms, work, s);
  return p.head_dim <= 64 ? launch<__nv_bfloat16, 64>(p, max_new, sms, work, s)
                          : launch<__nv_bfloat16, 128>(p, max_new, sms, work, s);
}

}  // namespace efg
