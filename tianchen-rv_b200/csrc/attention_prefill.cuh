// Attention of many query rows per request (prompts) over the paged Q4_0 cache, fp16 and bf16 calls: tcgen05
// products with their accumulators in tensor memory.
//
// A CTA takes 256 rows, two tiles of 128 (row = new token * heads of the kv head + head, so the heads that share a
// cache head share its tiles), and walks over the context in tiles of 128 tokens:
//   S = Q K^T (128 x 128, f32, TMEM)  ->  P = 2^(S * scale - m) (fp16, TMEM, over S)  ->  O += P V (128 x D, f32, TMEM).
// Warps 0..7 are the soft-max, of one tile after the other: two threads to a row, 64 columns each; warps 8..15 turn quants into the fp16
// operands in shared memory, warp 16 issues the products.  While one tile's soft-max runs the other tile's products do.
//
// What bounds it: the soft-max warps (a step of one tile takes them about 2100 SM cycles, 1024 of them the exponential unit's, and
// 2490 with keys whole, see below, for shared memory and issue slots are shared with twice the key operands); with values whole too
// 3070, the products of one tile no longer fitting behind the other's soft-max.  Besides its steps a CTA pays for its query rows, its
// first groups and its results, together as much as about eight pairs of steps when caches are cold.  4 prompts of up to 2048 tokens behind contexts of up
// to 2048, 32 / 8 heads of 128: bf16 450 us, 680 TFLOP/s of the pairs that count, with lse 510, fp16 567 (428 without second operands,
// 470 with the keys' alone).  Measured on the way, bf16 without second operands: four warps unpacking instead of eight 818 us; a thread
// to a row, one warpgroup to a tile, 459 (with the tiles' passes taking turns 510); half of the exponentials by a polynomial 517, for
// the schedulers have no cycles to spare for it.
//
// Numbers.  Key and value operands are d * (n - 8) rounded to fp16 (half a step of 2^-11), for their f32 sums could not be scaled
// block by block without reading S and O once for every block of 32.  What the rounding leaves out is a multiple of the scale's
// last place, hence an fp16 number: where an output shows it, it is a second operand whose product goes into the same sums.  So
//   fp16 results: keys and values whole (with both rounded, results were off by 1.7 times their own rounding);
//   bf16 results with lse, which is f32: keys whole (rounded, lse was off by 1e-4 over the root of the tokens seen);
//   bf16 results alone, whose own rounding is 8 times as large: both rounded.
// Query rows are fp16 after a power of two (exact for both types), weights are rounded to fp16; S, O, maximum and sum are f32.  A
// token with a scale so large that its values leave fp16 is held at 1/16 and made good in S or in P (its other blocks lose what lies
// below 2^-20).  The running maximum that P is relative to follows the true one only when that has grown by more than 2^8: then O is
// rescaled, otherwise P just has values up to 2^8.
#pragma once

#include <type_traits>

#include "attention_columns.cuh"
#include "tcgen05.cuh"

namespace tcrv {
namespace attention {

constexpr int kQuantWarps = 8;
constexpr int kProductWarp = 16;  // (the first of a warpgroup of which it alone has work)
constexpr int kPrefillThreads = 640;
// Registers: the block starts with 96 a thread; the soft-max takes over what the products' warpgroup can do without.
constexpr int kStartRegs = 96, kSoftmaxRegs = 136, kQuantRegs = 88, kProductRegs = 32;
static_assert(2 * kSoftmaxRegs + 2 * kQuantRegs + kProductRegs <= 5 * kStartRegs, "registers the block does not have");
constexpr int kTileRows = 128;
constexpr int kTileTokens = 128;
constexpr int kTileGroups = kTileTokens / kGroupTokens;
constexpr int kSlots = 4;  // tiles whose group flags are kept

struct PrefillParams {
  tcrv_cuda_attention_call call;
  uint32_t group;
  int32_t min_rows;      // requests with fewer rows (new tokens * group) are another kernel's
  int32_t splits;        // CTAs that share the tokens of one row block
  DeviceErrorWords errors;
};

// Workspace with splits > 1: (maximum, sum) and accumulators of each part's 256 rows.
__host__ __device__ inline size_t prefill_sums_offset(size_t parts) { return parts * 2 * kTileRows * 2 * sizeof(float); }
inline size_t prefill_workspace_bytes(size_t parts, size_t dim) {
  return prefill_sums_offset(parts) + parts * 2 * kTileRows * dim * sizeof(float);
}

// What the products see of keys and values.
constexpr int kRounded = 0;    // both rounded to fp16
constexpr int kExactKeys = 1;  // keys whole, as two terms with a product each
constexpr int kExactAll = 2;   // values too

template <int NB, int MODE>
struct PrefillLayout {
  static constexpr int kDim = 32 * NB;
  static constexpr int kPanel = 128 * 128;                       // 128 rows of 128 bytes
  static constexpr int kKeyBytes = kDim / 64 * kPanel;           // 128 tokens x D, K-major
  static constexpr int kValueBytes = kTileTokens / 64 * kDim * 128;  // D x 128 tokens, K-major
  static constexpr int kQuery = 0;
  static constexpr int kKeyStages = MODE == kExactAll ? 1 : 2;    // (what shared memory has room for)
  static constexpr int kKey = kQuery + 2 * kKeyBytes;
  static constexpr int kKeyLow = kKey + kKeyStages * kKeyBytes;   // second terms, one stage
  static constexpr int kValue = kKeyLow + (MODE != kRounded ? kKeyBytes : 0);
  static constexpr int kValueLow = kValue + 2 * kValueBytes;
  static constexpr int kFlags = kValueLow + (MODE == kExactAll ? kValueBytes : 0);  // u8 [slot][group]
  static constexpr int kPoison = kFlags + kSlots * kTileGroups;  // u16 [slot][group][block]: tokens whose value scale is no number
  static constexpr int kHeld = kPoison + kSlots * kTileGroups * NB * 2;     // u32 [slot][group]: tokens held at 1/16, keys, values << 16
  static constexpr int kBadRows = kHeld + kSlots * kTileGroups * 4;         // u8 [half][row]: blocks of which it sees such a token, tile 1's << 4
  static constexpr int kBars = kBadRows + 2 * 128;
  static constexpr int kBarCount = 24;
  static constexpr int kTops = kBars + kBarCount * 8;            // f32 [step parity][half][row]
  static constexpr int kTmem = kTops + 2 * 2 * 128 * 4;
  static constexpr int kAbort = kTmem + 4;
  static constexpr int kBytes = kAbort + 4;
  static_assert(kBytes <= 227 * 1024, "shared memory of a CTA");
  static_assert(NB <= 4 && kBars % 8 == 0, "blocks of a row in half a byte; barriers");
};

// barriers
enum { kBarQuery = 0, kBarKeyFull = 1, kBarKeyFree = 3, kBarValueFull = 5, kBarValueFree = 7, kBarScores = 9, kBarWeights = 11, kBarSums = 13, kBarPair = 15, kBarDrain = 19, kBarKeyLowFull = 20, kBarKeyLowFree = 21, kBarValueLowFull = 22, kBarValueLowFree = 23 };

// kind::f16, fp16 A and B (both K-major), f32 D.
__host__ __device__ constexpr uint32_t umma_idesc_f16(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// The upper half of umma_desc_k_major_sw128's descriptor does not depend on the address.
constexpr uint32_t kDescHigh = static_cast<uint32_t>((static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61) >> 32);
__device__ __forceinline__ uint32_t desc_low(uint32_t smem_byte_addr) { return ((smem_byte_addr & 0x3ffffu) >> 4) | (1u << 16); }
template <bool kAdd>
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %4};\n\t"
      "mov.b64 b, {%2, %4};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"
      "}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "n"(kDescHigh), "n"(kAdd ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 b;\n\t"
      "mov.b64 b, {%2, %4};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t"
      "}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "n"(kDescHigh), "r"(add)
      : "memory");
}

// v[0..16) into 16 consecutive columns of the warp's 32 lanes.
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// What quant * scale loses when it is rounded to fp16: exact, for it is a multiple of the scale's last place.
__device__ __forceinline__ uint32_t rounded_off(uint32_t quants, __half2 scale) {
  const __half2 n = bits_half2(quants);
  return half2_bits(__hfma2(n, scale, __hneg2(__hmul2(n, scale))));
}

// One lane's share of a group as it lies in the cache.
template <int NB>
struct RawGroup {
  uint32_t key[2][NB], value[2][NB];
  uint32_t key_scale[2][NB / 2];  // tokens g, g + 8
  uint32_t value_scale[2][NB];    // tokens (2t, 2t + 1), (2t + 8, 2t + 9)
  bool there;
};

template <int NB, int MODE>
__global__ void __launch_bounds__(kPrefillThreads, 1) prefill_kernel(const __grid_constant__ PrefillParams p) {
  using L = PrefillLayout<NB, MODE>;
  constexpr int kDim = L::kDim;
  extern __shared__ __align__(1024) uint8_t prefill_smem[];  // (the operands' swizzle goes by address bits; no room to round up)
  uint8_t *smem = prefill_smem;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBars);
  uint32_t *tmem_word = reinterpret_cast<uint32_t *>(smem + L::kTmem);
  volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(smem + L::kAbort);
  volatile uint8_t *flags = smem + L::kFlags;
  volatile uint16_t *poison = reinterpret_cast<volatile uint16_t *>(smem + L::kPoison);
  volatile uint32_t *held = reinterpret_cast<volatile uint32_t *>(smem + L::kHeld);
  volatile uint8_t *bad_rows = smem + L::kBadRows;
  const tcrv_cuda_attention_call &c = p.call;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_enter();
  if ((smem_addr(smem) & 1023u) != 0) {  // (never, as long as dynamic shared memory is given the alignment that it asks for)
    if (threadIdx.x == 0)
      raise_device_error(p.errors, kDevErrSharedAlignment);
    return;
  }
  // ---- what this CTA does: the longest row blocks come first
  const uint32_t kv_heads = static_cast<uint32_t>(c.cache.kv_heads);
  uint32_t id = blockIdx.x;
  const int part = static_cast<int>(id % p.splits);
  id /= p.splits;
  const uint32_t r = id % static_cast<uint32_t>(c.requests);
  id /= static_cast<uint32_t>(c.requests);
  const uint32_t head = id % kv_heads;
  const int32_t from_end = static_cast<int32_t>(id / kv_heads);
  const Request q = load_request(p.call, p.group, r, 1 << 30);
  const int32_t rows = q.rows * static_cast<int32_t>(p.group);
  const int32_t blocks = (rows + 2 * kTileRows - 1) / (2 * kTileRows);
  if (rows < p.min_rows || from_end >= blocks)
    return;
  const int32_t block = blocks - 1 - from_end, pair0 = block * 2 * kTileRows;
  const int tiles_q = rows - pair0 > kTileRows ? 2 : 1;
  const int32_t last_pair = min(rows, pair0 + 2 * kTileRows) - 1;
  const int32_t before = q.before;  // position of the request's first row
  const int32_t window = window_of(c);
  // the first token that the row at `position` sees, of those that there are
  const auto sees_from = [&](int32_t position) { return window ? max(0, max(-1, position) - window + 1) : 0; };
  const int32_t see_to = min(before + last_pair / static_cast<int32_t>(p.group), q.len - 1);  // the last row sees furthest
  const int32_t see_from = sees_from(before + pair0 / static_cast<int32_t>(p.group));
  int32_t tile_begin = see_from / kTileTokens, tile_end = see_to < see_from ? tile_begin : see_to / kTileTokens + 1;
  if (p.splits > 1) {
    const int32_t n = tile_end - tile_begin, b = tile_begin;
    tile_begin = b + static_cast<int32_t>(static_cast<int64_t>(n) * part / p.splits);
    tile_end = b + static_cast<int32_t>(static_cast<int64_t>(n) * (part + 1) / p.splits);
  }
  const int tiles = tile_end - tile_begin;

  if (threadIdx.x == 0) {
    mbar_init(&bars[kBarQuery], 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[kBarKeyFull + i], kQuantWarps);
      mbar_init(&bars[kBarKeyFree + i], 1);
      mbar_init(&bars[kBarValueFull + i], kQuantWarps);
      mbar_init(&bars[kBarValueFree + i], 1);
      mbar_init(&bars[kBarScores + i], 1);
      mbar_init(&bars[kBarWeights + i], 8);
      mbar_init(&bars[kBarSums + i], 1);
    }
    for (int i = 0; i < 4; ++i)
      mbar_init(&bars[kBarPair + i], 2);
    mbar_init(&bars[kBarDrain], 1);
    mbar_init(&bars[kBarKeyLowFull], kQuantWarps);
    mbar_init(&bars[kBarKeyLowFree], 1);
    mbar_init(&bars[kBarValueLowFull], kQuantWarps);
    mbar_init(&bars[kBarValueLowFree], 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kProductWarp) {
    tmem_alloc(tmem_word, 512);
    tmem_relinquish_alloc_permit();
  }
  tcgen05_fence_before_thread_sync();
  __syncthreads();
  tcgen05_fence_after_thread_sync();
  const uint32_t tmem = *tmem_word;
  // scores of tile i at columns 128 i (its weights over their first half), sums at 256 + D i
  const auto wait = [&](int bar, uint32_t parity) {
    if (mbar_wait_bounded(&bars[bar], parity & 1u, abort_flag))
      return true;
    if (*abort_flag == 0) {
      *abort_flag = 1;
      if (lane == 0)
        raise_device_error(p.errors, kDevErrBarrierTimeout);
    }
    return false;
  };

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ================================================================ soft-max of both tiles in turn
    // Two threads to a row, lane quadrant `warp & 3` and columns 64 * half .. + 63: the two warps of a scheduler then keep its
    // exponential unit busy together, and one tile's products run while the other tile's weights are made.
    const int half = warp >> 2, row0 = (warp & 3) * 32, row = row0 + lane;
    const uint32_t quadrant = static_cast<uint32_t>(row0) << 16;
    const int32_t group = static_cast<int32_t>(p.group);
    float *tops = reinterpret_cast<float *>(smem + L::kTops);
    int lifts = 0;  // powers of the queries of this thread's row in the two tiles, a byte each
    bad_rows[half * 128 + row] = 0;
    {
      // ---- the query operand, tile `half`: 32 rows of it, in the key operand's order of elements, times a power of two that
      // lifts the largest element into [2^14, 2^15).  kDim / 8 lanes to a row, eight elements to a lane.
      constexpr int kLanes = kDim / 8, kAtOnce = 32 / kLanes, kSteps = 32 / kAtOnce, kBatch = 8;
      uint8_t *operand = smem + L::kQuery + half * L::kKeyBytes;
      const int sub = lane % kLanes, b = sub >> 2, high = (sub >> 1) & 1, t = (sub & 1) * 2;
      const bool vector = (reinterpret_cast<uintptr_t>(c.q) & 15u) == 0 && ((c.q_row_stride | c.q_head_stride) & 7u) == 0;
      const float sign = c.scale < 0.0f ? -1.0f : 1.0f;
      int my_lift = 0;
#pragma unroll 1
      for (int s0 = 0; s0 < kSteps; s0 += kBatch) {
        uint4 raw[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int32_t pair = pair0 + half * kTileRows + row0 + (s0 + i) * kAtOnce + lane / kLanes, token = pair / group;
          raw[i] = make_uint4(0, 0, 0, 0);
          if (pair < rows) {
            const uint16_t *at = static_cast<const uint16_t *>(c.q) + static_cast<size_t>(q.first_row + token) * c.q_row_stride +
                                 (static_cast<size_t>(head) * group + (pair - token * group)) * c.q_head_stride + 8 * sub;
            if (vector) {
              raw[i] = *reinterpret_cast<const uint4 *>(at);
            } else {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = at[2 * e] | static_cast<uint32_t>(at[2 * e + 1]) << 16;
              raw[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
          float x[8], top = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (c.type == TCRV_CUDA_TYPE_F16) {
              const float2 f = __half22float2(bits_half2(w[e]));
              x[2 * e] = f.x, x[2 * e + 1] = f.y;
            } else {
              x[2 * e] = __uint_as_float(w[e] << 16), x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            }
            top = fmaxf(top, fmaxf(fabsf(x[2 * e]), fabsf(x[2 * e + 1])));
          }
#pragma unroll
          for (int off = kLanes / 2; off >= 1; off >>= 1)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          const int k = top > 0.0f && top < INFINITY ? min(120, 141 - static_cast<int>(__float_as_uint(top) >> 23)) : 0;
          const float lift = __uint_as_float(static_cast<uint32_t>(127 + k) << 23) * sign;
          const int line_row = row0 + (s0 + i) * kAtOnce + lane / kLanes;
#pragma unroll
          for (int h = 0; h < kAtOnce; ++h) {  // lane `row` keeps the row's power
            const int its = __shfl_sync(0xffffffffu, k, h * kLanes);
            if (lane == (s0 + i) * kAtOnce + h)
              my_lift = its;
          }
          uint8_t *line = operand + (b >> 1) * L::kPanel + line_row * 128 + high * 8;
#pragma unroll
          for (int u = 0; u < 2; ++u) {  // elements 4t', 4t'+2, 4t'+1, 4t'+3 of the half block
            const int chunk = 2 * (t + u) + (b & 1);
            const uint2 v = make_uint2(half2_bits(__floats2half2_rn(x[4 * u] * lift, x[4 * u + 2] * lift)),
                                       half2_bits(__floats2half2_rn(x[4 * u + 1] * lift, x[4 * u + 3] * lift)));
            *reinterpret_cast<uint2 *>(line + ((chunk ^ (line_row & 7)) << 4)) = v;
          }
        }
      }
      // the row's power in the other tile is the other warp's
      reinterpret_cast<int *>(tops)[half * 128 + row] = my_lift;
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars[kBarQuery]);
        mbar_arrive(&bars[kBarPair + (warp & 3)]);
      }
      if (wait(kBarPair + (warp & 3), 0)) {
        const int other = reinterpret_cast<int *>(tops)[(1 - half) * 128 + row];
        lifts = half == 0 ? (my_lift & 0xff) | other << 8 : (other & 0xff) | my_lift << 8;
      }
    }
    // what changes between the tiles; the loop below swaps `mine` and `other` after each step
    struct State {
      float m, l, scale;
      int32_t position, from, to;  // what this row sees up to; tokens that all rows of the tile see
    };
    const auto state_of = [&](int tile, int lift) {
      const int32_t pair = pair0 + tile * kTileRows + row;
      State st;
      st.position = pair < rows ? max(-1, before + pair / group) : -1;
      // (a row that sees nothing has a maximum, so that it does not hold up its warp)
      st.m = st.position < 0 ? 0.0f : -INFINITY;
      st.l = 0.0f;
      st.scale = fabsf(c.scale) * kLog2e * __uint_as_float(static_cast<uint32_t>(127 - lift) << 23);
      const int32_t first = pair0 + tile * kTileRows;
      st.from = sees_from(before + (min(rows, first + kTileRows) - 1) / group);
      st.to = max(-1, before + first / group) - (kTileTokens - 1);
      return st;
    };
    State mine = state_of(0, static_cast<int8_t>(lifts)), other = state_of(1, static_cast<int8_t>(lifts >> 8));
    const int steps = tiles * tiles_q;
#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
      const int tile = tiles_q == 2 ? step & 1 : 0, j = tiles_q == 2 ? step >> 1 : step;
      if (!wait(kBarScores + tile, j))
        break;
      tcgen05_fence_after_thread_sync();
      const uint32_t scores = tmem + quadrant + tile * 128, sums = tmem + quadrant + 256 + tile * kDim;
      uint32_t s[64], w[32];
      tmem_ld_32x32b<32>(scores + half * 64, *reinterpret_cast<uint32_t(*)[32]>(s));
      tmem_ld_32x32b<32>(scores + half * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
      const int32_t token0 = (tile_begin + j) * kTileTokens;
      const int slot = j % kSlots;
      const uint64_t group_flags = *reinterpret_cast<volatile uint64_t *>(smem + L::kFlags + slot * kTileGroups);
      const bool whole = group_flags == 0x0101010101010101ull && token0 >= mine.from && token0 <= mine.to;
      // columns that this row sees
      const int32_t upper = mine.position - token0 - half * 64, lower = window && window <= upper ? upper - window + 1 : 0;
      if (!whole) {  // scores in powers of two, unseen ones -infinity; the weights' scale is 1 then
        tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const uint32_t flag = static_cast<uint32_t>(group_flags >> (8 * (4 * half + h)));
          if (flag & 2u) {  // keys held at 1/16
            const uint32_t keys = held[slot * kTileGroups + 4 * half + h];
#pragma unroll
            for (int i = 0; i < kGroupTokens; ++i)
              s[16 * h + i] = (keys >> i) & 1u ? __float_as_uint(16.0f * __uint_as_float(s[16 * h + i])) : s[16 * h + i];
          }
          const int32_t to = (flag & 1u) ? upper : -1;
#pragma unroll
          for (int i = 16 * h; i < 16 * h + 16; ++i)
            s[i] = i <= to && i >= lower ? __float_as_uint(__uint_as_float(s[i]) * mine.scale) : 0xff800000u;
        }
      }
      const float by = whole ? mine.scale : 1.0f;
      // Weights relative to the maximum of the tiles before, which is as good as this tile's own unless that is more than 2^8
      // above it (or there is none yet): then the accumulators are rescaled and the weights made again.
      tmem_ld_wait();
      float top;
      {
        float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 64; i += 2)
          most[(i >> 1) & 3] = max3(most[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * by;
      }
      // to the thread that has the row's other half; its maximum is here by the time the weights are made
      float *exchange = tops + ((step + 1) & 1) * 256;  // (the prologue's was the first)
      exchange[half * 128 + row] = top;
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&bars[kBarPair + (warp & 3)]);
      float2 parts[2];
      const auto weigh = [&](float base) {
        const float2 by2 = make_float2(by, by), base2 = make_float2(-base, -base);
        parts[0] = parts[1] = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          float2 x = fma2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), by2, base2);
          x.x = exp2_fast(x.x);
          x.y = exp2_fast(x.y);
          parts[(i >> 1) & 1] = add2(parts[(i >> 1) & 1], x);
          w[i / 2] = half2_bits(__floats2half2_rn(x.x, x.y));
        }
      };
      if (j > 0)
        weigh(mine.m == -INFINITY ? 0.0f : mine.m);
      if (!wait(kBarPair + (warp & 3), step + 1))
        break;
      top = fmaxf(top, exchange[(1 - half) * 128 + row]);
      const bool grown = top > mine.m + 8.0f || (mine.m == -INFINITY && top > -INFINITY);
      if (__any_sync(0xffffffffu, grown || j == 0)) {
        const float now = grown ? top : mine.m, alpha = grown ? exp2_fast(mine.m - now) : 1.0f;
        mine.m = now;
        mine.l *= alpha;
        if (j > 0) {
          if (!wait(kBarSums + tile, j - 1))
            break;
          tcgen05_fence_after_thread_sync();
#pragma unroll 1
          for (int ch = 0; ch < kDim / 32; ++ch) {
            uint32_t o[16];
            const uint32_t at = sums + half * (kDim / 2) + ch * 16;
            tmem_ld_32x32b<16>(at, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i)
              o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st_32x32b_x16(at, o);
          }
        }
        weigh(mine.m == -INFINITY ? 0.0f : mine.m);
      }
      mine.l += (parts[0].x + parts[0].y) + (parts[1].x + parts[1].y);
      if (!whole && group_flags != 0x0101010101010101ull) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const uint32_t flag = static_cast<uint32_t>(group_flags >> (8 * (4 * half + h)));
          if (flag & 4u) {  // values held at 1/16
            const uint32_t values = held[slot * kTileGroups + 4 * half + h] >> 16;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              w[8 * h + i] = half2_bits(__hmul2(bits_half2(w[8 * h + i]), __floats2half2_rn((values >> (2 * i)) & 1u ? 16.0f : 1.0f, (values >> (2 * i)) & 2u ? 16.0f : 1.0f)));
          }
          if (flag & 8u) {  // values that are no numbers: nor are the elements of their block, of the rows that see their token
            const int32_t first = max(lower - 16 * h, 0), last = min(upper - 16 * h, kGroupTokens - 1);
            const uint32_t seen = first <= last ? (2u << last) - (1u << first) : 0u;
            uint32_t blocks = 0;
#pragma unroll
            for (int b = 0; b < NB; ++b)
              blocks |= (poison[(slot * kTileGroups + 4 * half + h) * NB + b] & seen) ? 1u << b : 0u;
            if (blocks)
              bad_rows[half * 128 + row] |= static_cast<uint8_t>(blocks << (4 * tile));
          }
        }
      }
      tmem_st_32x32b_x16(scores + half * 32, *reinterpret_cast<const uint32_t(*)[16]>(w));
      tmem_st_32x32b_x16(scores + half * 32 + 16, *reinterpret_cast<const uint32_t(*)[16]>(w + 16));
      tmem_st_wait();
      tcgen05_fence_before_thread_sync();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&bars[kBarWeights + tile]);
      if (tiles_q == 2) {
        const State swap = mine;
        mine = other;
        other = swap;
      }
    }
    // ---- the rows' results, each thread half of the elements; element n of the sums is
    // d = 32 (n / 32) + 16 ((n >> 4) & 1) + 2 (n & 7) + ((n >> 3) & 1)
    const bool vector = (reinterpret_cast<uintptr_t>(c.out) & 15u) == 0 && ((c.out_row_stride | c.out_head_stride) & 7u) == 0;
#pragma unroll 1
    for (int tile = 0; tile < tiles_q; ++tile) {
      const State &st = tile == 0 ? mine : other;
      bool done = tiles > 0 && *abort_flag == 0;
      if (done) {
        done = wait(kBarSums + tile, tiles - 1);
        tcgen05_fence_after_thread_sync();
      }
      // the row's sum is in two threads
      float *exchange = tops + ((steps + tile + 1) & 1) * 256;
      exchange[half * 128 + row] = st.l;
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&bars[kBarPair + (warp & 3)]);
      float l = st.l;
      if (wait(kBarPair + (warp & 3), steps + 1 + tile))
        l = half == 0 ? l + exchange[128 + row] : exchange[row] + l;
      const uint32_t bad = static_cast<uint32_t>(bad_rows[row] | bad_rows[128 + row]) >> (4 * tile);
      const int32_t pair = pair0 + tile * kTileRows + row, token = pair / group;
      const size_t q_head = static_cast<size_t>(head) * group + (pair - token * group);
      const size_t at = static_cast<size_t>(q.first_row + token) * c.out_row_stride + q_head * c.out_head_stride;
      const size_t slot = (static_cast<size_t>(blockIdx.x) * 2 + tile) * kTileRows + row;
      float *part_sums = p.splits > 1 ? reinterpret_cast<float *>(static_cast<uint8_t *>(c.workspace) + prefill_sums_offset(gridDim.x)) + slot * kDim : nullptr;
      const bool any = done && (l > 0.0f || l != l);
      const float factor = !any ? 0.0f : p.splits > 1 ? 1.0f : 1.0f / l;
#pragma unroll 1
      for (int b = half * (NB / 2); b < (half + 1) * (NB / 2); ++b) {
        uint32_t o[32];
        tmem_ld_32x32b<32>(tmem + quadrant + 256 + tile * kDim + b * 32, o);
        tmem_ld_wait();
        float y[32];
#pragma unroll
        for (int d = 0; d < 32; ++d) {
          const float v = __uint_as_float(o[(d >> 4) * 16 + (d & 1) * 8 + ((d & 15) >> 1)]);
          y[d] = (bad >> b) & 1u ? NAN : any ? v * factor : 0.0f;  // (without a product the columns hold anything)
        }
        if (pair < rows) {
          if (part_sums != nullptr) {
#pragma unroll
            for (int d = 0; d < 32; d += 4)
              *reinterpret_cast<float4 *>(part_sums + b * 32 + d) = make_float4(y[d], y[d + 1], y[d + 2], y[d + 3]);
          } else if (vector) {
#pragma unroll
            for (int d = 0; d < 32; d += 8) {
              uint32_t v[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (c.type == TCRV_CUDA_TYPE_F16) {
                  v[i] = half2_bits(__floats2half2_rn(y[d + 2 * i], y[d + 2 * i + 1]));
                } else {
                  const __nv_bfloat162 h = __floats2bfloat162_rn(y[d + 2 * i], y[d + 2 * i + 1]);
                  memcpy(&v[i], &h, 4);
                }
              }
              *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(c.out) + at + b * 32 + d) = make_uint4(v[0], v[1], v[2], v[3]);
            }
          } else {
#pragma unroll
            for (int d = 0; d < 32; ++d)
              store_typed(c.out, at + b * 32 + d, c.type, y[d]);
          }
        }
      }
      if (pair < rows && half == 0) {
        if (part_sums != nullptr)
          *reinterpret_cast<float2 *>(static_cast<float *>(c.workspace) + slot * 2) = make_float2(st.m, done ? l : 0.0f);
        else if (c.lse != nullptr)
          c.lse[static_cast<size_t>(q.first_row + token) * c.heads + q_head] = any ? (st.m + log2f(l)) * 0.6931471805599453f : -INFINITY;
      }
    }
  } else if (warp < kProductWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kQuantRegs));
    // ================================================================ quants -> fp16 operands
    // a warp to each group of a tile
    const int w = warp - 8, g = lane >> 2, t = lane & 3;
    const int32_t per_page = static_cast<int32_t>(c.cache.groups);
    const int32_t groups = (q.len + kGroupTokens - 1) / kGroupTokens;
    const int32_t *table = c.block_table + r * c.table_stride;
    // the group whose page is asked for next, and its place in its page
    int32_t at = tile_begin * kTileGroups + w, page_at = at / per_page, in_page = at - page_at * per_page, page = -1, place = 0;
    const int32_t end = min(groups, tile_end * kTileGroups);
    const auto ask = [&]() {
      page = at < end ? table[page_at] : -1;
      place = in_page;
      at += kTileGroups;
      in_page += kTileGroups;
      while (in_page >= per_page) {
        in_page -= per_page;
        ++page_at;
      }
    };
    const auto fetch = [&](RawGroup<NB> &raw) {
      raw.there = page >= 0 && static_cast<size_t>(page) < c.cache.pages;
      if (raw.there) {
        // (ordinary loads: the read-only path is for memory that nobody writes while the kernel lives, and its life may begin
        // while the call before it still fills the cache)
        const uint8_t *from = c.cache.data + static_cast<size_t>(page) * c.cache.page_stride +
                              (static_cast<size_t>(head) * per_page + place) * (18 * kDim);
        load_words<NB>(raw.key[0], from + lane * NB * 4);
        load_words<NB>(raw.key[1], from + 128 * NB + lane * NB * 4);
        load_words<NB>(raw.value[0], from + 256 * NB + lane * NB * 4);
        load_words<NB>(raw.value[1], from + 384 * NB + lane * NB * 4);
        load_words<NB / 2>(raw.key_scale[0], from + 512 * NB + g * NB * 2);
        load_words<NB / 2>(raw.key_scale[1], from + 512 * NB + (g + 8) * NB * 2);
        load_words<NB>(raw.value_scale[0], from + 544 * NB + 2 * t * NB * 2);
        load_words<NB>(raw.value_scale[1], from + 544 * NB + (2 * t + 8) * NB * 2);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int b = 0; b < NB; ++b)
            raw.key[h][b] = raw.value[h][b] = raw.value_scale[h][b] = 0;
#pragma unroll
          for (int b = 0; b < NB / 2; ++b)
            raw.key_scale[h][b] = 0;
        }
      }
    };
    // this lane's places in the operands; neighbouring lanes' chunks fall on different banks
    uint8_t *const key_even = smem + L::kKey + (w * kGroupTokens + g) * 128 + (((2 * t) ^ g) << 4);
    uint8_t *const key_odd = smem + L::kKey + (w * kGroupTokens + g) * 128 + (((2 * t + 1) ^ g) << 4);
    uint8_t *const value_first = smem + L::kValue + (w >> 2) * (kDim * 128) + g * 128 + t * 4 + ((((w & 3) * 2) ^ g) << 4);
    uint8_t *const value_second = smem + L::kValue + (w >> 2) * (kDim * 128) + g * 128 + t * 4 + ((((w & 3) * 2 + 1) ^ g) << 4);
    const auto convert = [&](RawGroup<NB> &now, int j) -> bool {
      const int stage = j & 1, key_stage = j % L::kKeyStages, slot = j % kSlots;
      // ---- scales: of values, two tokens side by side; none for tokens behind the context; large ones are seen to
      uint32_t pair[2][NB];
      uint32_t some = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          pair[h][b] = __byte_perm(now.value_scale[h][b / 2], now.value_scale[h][NB / 2 + b / 2], (b & 1) ? 0x7632 : 0x5410);
          some |= now.value_scale[h][b];
        }
#pragma unroll
        for (int b = 0; b < NB / 2; ++b)
          some |= now.key_scale[h][b];
      }
      const int32_t left = q.len - ((tile_begin + j) * kTileGroups + w) * kGroupTokens;
      if (left < kGroupTokens) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t keep = (2 * t + 8 * h < left ? 0xffffu : 0u) | (2 * t + 8 * h + 1 < left ? 0xffff0000u : 0u);
#pragma unroll
          for (int b = 0; b < NB; ++b)
            pair[h][b] &= keep;
#pragma unroll
          for (int b = 0; b < NB / 2; ++b)
            now.key_scale[h][b] = g + 8 * h < left ? now.key_scale[h][b] : 0;
        }
      }
      uint32_t flag = now.there ? 1u : 0u;
      // A scale of 2^13 or more (8 d may leave fp16), an infinity or a NaN has these three bits; so may several others together.  Then
      // the tokens that have one are looked for and held at 1/16, which others of the group would not bear (below 2^-10 a sixteenth is
      // not exact).
      if (__any_sync(0xffffffffu, (some & 0x7000u) == 0x7000u || (some & 0x70000000u) == 0x70000000u)) {
        uint32_t bad[NB] = {}, any_bad = 0, large = 0;  // large: keys' tokens, values' << 16
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const uint32_t d = (b & 1) ? now.key_scale[h][b / 2] >> 16 : now.key_scale[h][b / 2];
            large |= (d & 0x7000u) == 0x7000u ? 1u << (g + 8 * h) : 0u;
            if ((pair[h][b] & 0x7c00u) == 0x7c00u) {
              bad[b] |= 1u << (2 * t + 8 * h);
              pair[h][b] &= 0xffff0000u;
            }
            if ((pair[h][b] & 0x7c000000u) == 0x7c000000u) {
              bad[b] |= 2u << (2 * t + 8 * h);
              pair[h][b] &= 0xffffu;
            }
            large |= (pair[h][b] & 0x7000u) == 0x7000u ? 0x10000u << (2 * t + 8 * h) : 0u;
            large |= (pair[h][b] & 0x70000000u) == 0x70000000u ? 0x20000u << (2 * t + 8 * h) : 0u;
          }
        }
        large = __reduce_or_sync(0xffffffffu, large);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const __half2 key_by = __float2half2_rn((large >> (g + 8 * h)) & 1u ? 0.0625f : 1.0f);
          const uint32_t two = large >> (16 + 2 * t + 8 * h);
          const __half2 value_by = __floats2half2_rn(two & 1u ? 0.0625f : 1.0f, two & 2u ? 0.0625f : 1.0f);
#pragma unroll
          for (int b = 0; b < NB / 2; ++b)
            now.key_scale[h][b] = half2_bits(__hmul2(bits_half2(now.key_scale[h][b]), key_by));
#pragma unroll
          for (int b = 0; b < NB; ++b)
            pair[h][b] = half2_bits(__hmul2(bits_half2(pair[h][b]), value_by));
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          bad[b] = __reduce_or_sync(0xffffffffu, bad[b]);
          any_bad |= bad[b];
          if (lane == 0)
            poison[(slot * kTileGroups + w) * NB + b] = static_cast<uint16_t>(bad[b]);
        }
        if (lane == 0)
          held[slot * kTileGroups + w] = large;
        flag |= (large & 0xffffu ? 2u : 0u) | (large >> 16 ? 4u : 0u) | (any_bad ? 8u : 0u);
      }
      if (j >= L::kKeyStages && !wait(kBarKeyFree + key_stage, j / L::kKeyStages - 1))
        return false;
      if (lane == 0)
        flags[slot * kTileGroups + w] = static_cast<uint8_t>(flag);
      // ---- keys: a word's 8 elements are 16 bytes of the token's row
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint32_t word = now.key[h][b];
          const __half2 scale = bits_half2(__byte_perm(now.key_scale[h][b / 2], 0, (b & 1) ? 0x3232 : 0x1010));
          const uint4 v = make_uint4(half2_bits(__hmul2(bits_half2(low_nibbles(word)), scale)),
                                     half2_bits(__hmul2(bits_half2(low_nibbles(word >> 8)), scale)),
                                     half2_bits(__hmul2(bits_half2(high_nibbles(word)), scale)),
                                     half2_bits(__hmul2(bits_half2(high_nibbles(word >> 8)), scale)));
          *reinterpret_cast<uint4 *>(((b & 1) ? key_odd : key_even) + key_stage * L::kKeyBytes + (b >> 1) * L::kPanel + h * 1024) = v;
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&bars[kBarKeyFull + key_stage]);
      // ---- what the fp16 keys leave out
      if constexpr (MODE != kRounded) {
        if (j >= 1 && !wait(kBarKeyLowFree, j - 1))
          return false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            uint32_t word = now.key[h][b];
            asm volatile("" : "+r"(word));  // (unpacked again: kept from above, it would take 32 registers)
            const __half2 scale = bits_half2(__byte_perm(now.key_scale[h][b / 2], 0, (b & 1) ? 0x3232 : 0x1010));
            const uint4 v = make_uint4(rounded_off(low_nibbles(word), scale), rounded_off(low_nibbles(word >> 8), scale),
                                       rounded_off(high_nibbles(word), scale), rounded_off(high_nibbles(word >> 8), scale));
            *reinterpret_cast<uint4 *>(((b & 1) ? key_odd : key_even) + (L::kKeyLow - L::kKey) + (b >> 1) * L::kPanel + h * 1024) = v;
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&bars[kBarKeyLowFull]);
      }
      // ---- values, transposed: row n of the operand is an element, its columns the tokens
      if (j >= 2 && !wait(kBarValueFree + stage, (j >> 1) - 1))
        return false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint32_t word = now.value[h][b];
          const __half2 scale = bits_half2(pair[h][b]);
          const uint32_t v[4] = {half2_bits(__hmul2(bits_half2(low_nibbles(word)), scale)),
                                 half2_bits(__hmul2(bits_half2(low_nibbles(word >> 8)), scale)),
                                 half2_bits(__hmul2(bits_half2(high_nibbles(word)), scale)),
                                 half2_bits(__hmul2(bits_half2(high_nibbles(word >> 8)), scale))};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<uint32_t *>((h ? value_second : value_first) + stage * L::kValueBytes + (b * 4 + k) * 1024) = v[k];
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&bars[kBarValueFull + stage]);
      // ---- what the fp16 values leave out
      if constexpr (MODE == kExactAll) {
        if (j >= 1 && !wait(kBarValueLowFree, j - 1))
          return false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            uint32_t word = now.value[h][b];
            asm volatile("" : "+r"(word));
            const __half2 scale = bits_half2(pair[h][b]);
            const uint32_t v[4] = {rounded_off(low_nibbles(word), scale), rounded_off(low_nibbles(word >> 8), scale),
                                   rounded_off(high_nibbles(word), scale), rounded_off(high_nibbles(word >> 8), scale)};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *reinterpret_cast<uint32_t *>((h ? value_second : value_first) + (L::kValueLow - L::kValue) + (b * 4 + k) * 1024) = v[k];
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&bars[kBarValueLowFull]);
      }
      return true;
    };
    // Two tiles' groups are on their way; each register set is filled again as soon as it has been used, without a copy.
    RawGroup<NB> even, odd;
    ask();
    fetch(even);
    ask();
    fetch(odd);
    ask();
#pragma unroll 1
    for (int j = 0; j < tiles; j += 2) {
      if (!convert(even, j))
        break;
      fetch(even);
      ask();
      if (j + 1 >= tiles || !convert(odd, j + 1))
        break;
      fetch(odd);
      ask();
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProductRegs));
    if (warp == kProductWarp && tiles > 0) {
    // ================================================================ products: one lane issues
    // (values that the compiler knows to be the same in every lane go to the instruction without a detour)
    const uint32_t base = __shfl_sync(0xffffffffu, smem_addr(smem), 0), columns = __shfl_sync(0xffffffffu, tmem, 0);
    constexpr uint32_t kScoreDesc = umma_idesc_f16(kTileRows, kTileTokens), kSumDesc = umma_idesc_f16(kTileRows, kDim);
    const bool leader = elect_one();
    // (second terms first: their place is free soonest)
    const auto score = [&](int tile, int stage, bool last) {
      const uint32_t a = desc_low(base + L::kQuery + tile * L::kKeyBytes), b = desc_low(base + L::kKey + stage * L::kKeyBytes);
      if constexpr (MODE != kRounded) {
        const uint32_t low = desc_low(base + L::kKeyLow);
        umma_f16_ss<false>(columns + tile * 128, a, low, kScoreDesc);
#pragma unroll
        for (int k = 1; k < kDim / 16; ++k) {
          const uint32_t at = (k / 4) * (L::kPanel >> 4) + (k % 4) * 2;
          umma_f16_ss<true>(columns + tile * 128, a + at, low + at, kScoreDesc);
        }
        if (last)
          umma_commit(&bars[kBarKeyLowFree]);
      }
      umma_f16_ss<MODE != kRounded>(columns + tile * 128, a, b, kScoreDesc);
#pragma unroll
      for (int k = 1; k < kDim / 16; ++k) {
        const uint32_t at = (k / 4) * (L::kPanel >> 4) + (k % 4) * 2;
        umma_f16_ss<true>(columns + tile * 128, a + at, b + at, kScoreDesc);
      }
      umma_commit(&bars[kBarScores + tile]);
      if (last)
        umma_commit(&bars[kBarKeyFree + stage]);
    };
    const auto sum = [&](int tile, int stage, bool add, bool last) {
      const uint32_t b = desc_low(base + L::kValue + stage * L::kValueBytes);
      if constexpr (MODE == kExactAll) {
        const uint32_t low = desc_low(base + L::kValueLow);
#pragma unroll
        for (int k = 0; k < kTileTokens / 16; ++k) {
          const uint32_t at = (k / 4) * ((kDim * 128) >> 4) + (k % 4) * 2;
          umma_f16_ts(columns + 256 + tile * kDim, columns + tile * 128 + k * 8, low + at, kSumDesc, k > 0 || add ? 1u : 0u);
        }
        if (last)
          umma_commit(&bars[kBarValueLowFree]);
        add = true;
      }
#pragma unroll
      for (int k = 0; k < kTileTokens / 16; ++k) {
        const uint32_t at = (k / 4) * ((kDim * 128) >> 4) + (k % 4) * 2;
        umma_f16_ts(columns + 256 + tile * kDim, columns + tile * 128 + k * 8, b + at, kSumDesc, k > 0 || add ? 1u : 0u);
      }
      umma_commit(&bars[kBarSums + tile]);
      if (last)
        umma_commit(&bars[kBarValueFree + stage]);
    };
    bool good = wait(kBarQuery, 0) && wait(kBarKeyFull, 0) && (MODE == kRounded || wait(kBarKeyLowFull, 0));
    tcgen05_fence_after_thread_sync();
    if (good && leader) {
      for (int i = 0; i < tiles_q; ++i)
        score(i, 0, i == tiles_q - 1);
    }
#pragma unroll 1
    for (int j = 0; j < tiles && good; ++j) {
      const int next = (j + 1) % L::kKeyStages;
      good = wait(kBarValueFull + (j & 1), j >> 1) && (MODE != kExactAll || wait(kBarValueLowFull, j));
      for (int i = 0; i < tiles_q && good; ++i) {
        good = wait(kBarWeights + i, j);
        tcgen05_fence_after_thread_sync();
        if (good && leader)
          sum(i, j & 1, j > 0, i == tiles_q - 1);
        __syncwarp();
        if (j + 1 < tiles) {
          if (i == 0 && good)
            good = wait(kBarKeyFull + next, (j + 1) / L::kKeyStages) && (MODE == kRounded || wait(kBarKeyLowFull, j + 1));
          tcgen05_fence_after_thread_sync();
          if (good && leader)
            score(i, next, i == tiles_q - 1);
          __syncwarp();
        }
      }
    }
    if (!good) {  // products on their way end before their memory goes back
      if (leader)
        umma_commit(&bars[kBarDrain]);
      __syncwarp();
      mbar_wait_bounded(&bars[kBarDrain], 0);
    }
    }
  }
  // ---- the tensor memory goes back when every role is through with it
  tcgen05_fence_before_thread_sync();
  __syncthreads();
  tcgen05_fence_after_thread_sync();
  if (warp == kProductWarp)
    tmem_dealloc(tmem, 512);
}

// Joins the parts of a row block: one warp per row.
template <int NB>
__global__ void __launch_bounds__(256) prefill_combine_kernel(const __grid_constant__ PrefillParams p, uint32_t parts) {
  constexpr int kDim = 32 * NB;
  pdl_enter();
  const tcrv_cuda_attention_call &c = p.call;
  const uint32_t kv_heads = static_cast<uint32_t>(c.cache.kv_heads);
  const int lane = threadIdx.x & 31;
  uint32_t id = blockIdx.y;
  const uint32_t first_part = id * p.splits;
  const uint32_t r = id % static_cast<uint32_t>(c.requests);
  id /= static_cast<uint32_t>(c.requests);
  const uint32_t head = id % kv_heads;
  const int32_t from_end = static_cast<int32_t>(id / kv_heads);
  const Request q = load_request(p.call, p.group, r, 1 << 30);
  const int32_t rows = q.rows * static_cast<int32_t>(p.group), blocks = (rows + 2 * kTileRows - 1) / (2 * kTileRows);
  if (rows < p.min_rows || from_end >= blocks)
    return;
  const int32_t pair0 = (blocks - 1 - from_end) * 2 * kTileRows, row = static_cast<int32_t>(blockIdx.x * 8 + (threadIdx.x >> 5)), pair = pair0 + row;
  if (pair >= rows)
    return;
  const float2 *stats = static_cast<const float2 *>(c.workspace);
  const float *sums = reinterpret_cast<const float *>(static_cast<const uint8_t *>(c.workspace) + prefill_sums_offset(parts));
  const auto slot = [&](int i) { return (static_cast<size_t>(first_part + i) * 2 * kTileRows) + row; };
  float top = -INFINITY;
  for (int i = 0; i < p.splits; ++i)
    top = fmaxf(top, stats[slot(i)].x);
  const float base = top == -INFINITY ? 0.0f : top;
  float total = 0.0f, sum[NB] = {};
  for (int i = 0; i < p.splits; ++i) {
    const float2 ml = stats[slot(i)];
    const float f = exp2_fast(ml.x - base);
    total = fmaf(f, ml.y, total);
#pragma unroll
    for (int b = 0; b < NB; ++b)
      sum[b] = fmaf(f, sums[slot(i) * kDim + b * 32 + lane], sum[b]);
  }
  const int32_t token = pair / static_cast<int32_t>(p.group);
#pragma unroll
  for (int b = 0; b < NB; ++b)
    write_row(c, q.first_row + token, head * p.group + (pair - token * p.group), b * 32 + lane, sum[b], total, top);
}

}  // namespace attention
}  // namespace tcrv
