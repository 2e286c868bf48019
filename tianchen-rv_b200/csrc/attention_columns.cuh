// Attention of a few query rows per request over the paged Q4_0 cache (decode, drafted tokens, and
// every call whose rows need more than fp16 products): the context's tokens are the M side of the
// tensor cores' m16n8k16 product and the query rows its N side,
//   S^T[token][row] = K q^T        and        O^T[d][row] = V^T P^T,
// so eight rows fill a tile that the other way round would be half empty, and a key or value operand is
// used as it lies in the cache (kv_layout.cuh): one AND with a mask turns a word into a register of the
// operand.
//
// Numbers.  A cached value is d * (n - 8).  Its integer part is exact in fp16 and the products with it are
// summed in f32; the scales stay outside: the key's multiplies the f32 sum over its block, the value's
// multiplies the soft-max weight, one operand per block.  What is rounded is the query row (scaled by a
// power of two so that its largest element lies in [2^14, 2^15)) and the weight times the value's scale
// (lifted by a power of two that brings the largest scale seen so far into [2^14, 2^15)):
//   fp16 and bf16 calls: both to one fp16 term, half a step of 2^-11 (a 16-bit query is exact);
//   f32 calls: both to two fp16 terms, 2^-22 relative, with a product each into the same sums, or up to 4
//   rows with a column each (4 rows, cold caches: 777 tokens 19.5 us against 15.4, 64 x 2048 tokens 87 against 65).
// A weight times its scale leaves fp16's normal range below 2^-28 of the largest scale: what it then loses is at most 2^-39 of that
// scale.  (Without a lift values of 1e-4 lost a percent, and those beside a token e^8 above them more.)
// Maximum, sum and accumulators are f32.
#pragma once

#include "async_copy.cuh"
#include "kv_layout.cuh"

namespace tcrv {
namespace attention {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kUnitGroups = 2;                             // groups of 16 tokens to a warp's step
constexpr int kUnitTokens = kUnitGroups * kGroupTokens;
constexpr int kCombineThreads = 128;
// What the end of a segment costs a CTA, in units: its warps wait for the last of them and join their parts.  Counted into the
// list that is cut into ranges, or the CTAs among short contexts end last.  With 8, 20 and 40, us, cold caches: 64 requests of up to
// 8191 tokens, bf16, heads of 64: 91, 87, 91, of 128: 132, 122, 128, of 256: 247, 216, 218, f32 114, 110, 114; 16 x 5 drafted tokens,
// f32: 87, 79, 85, bf16: 83, 75, 77.
constexpr int kSegmentUnits = 20;
constexpr float kLog2e = 1.4426950408889634f;

struct ColumnParams {
  tcrv_cuda_attention_call call;
  uint32_t group;       // query heads to a kv head
  long long most_rows;  // requests with more rows (new tokens * group) are another kernel's
  DeviceErrorWords errors;
};

// What the combine step has to know of the context range that begins in CTA c and ends in a later one.
struct SplitRange {
  int32_t valid, head, column_group, last_cta, rows, first_row;
  int32_t pad[2];
};

// Workspace: one SplitRange per CTA, then (maximum, sum) and the accumulators of two partial ranges per
// CTA (the one that began before it, the one that ends after it).
__host__ __device__ inline size_t column_stats_offset(size_t ctas) { return ctas * sizeof(SplitRange); }
__host__ __device__ inline size_t column_sums_offset(size_t ctas, size_t rows) {
  return column_stats_offset(ctas) + 2 * ctas * rows * 2 * sizeof(float);
}
inline size_t column_workspace_bytes(size_t ctas, size_t rows, size_t dim) {
  return column_sums_offset(ctas, rows) + 2 * ctas * rows * dim * sizeof(float);
}

inline int ctas_per_sm(int nb, int nt) { return nb * nt <= 4 ? 2 : 1; }

// How a call's numbers become fp16 operands.
constexpr int kOneTerm = 1;   // fp16 and bf16
constexpr int kTwoTerms = 2;  // f32: two products into the same sums
constexpr int kPairs = 3;     // f32, up to 4 rows: the terms in neighbouring columns of the one tile, which has room for them

template <int NB, int NT, int MODE>
struct ColumnLayout {
  static constexpr int kDim = 32 * NB;
  static constexpr int kStages = NB * NT <= 2 ? 4 : NB * NT <= 3 ? 3 : NB >= 6 ? 2 : NB * NT > 4 ? 4 : 2;  // (what shared memory has room for)
  static constexpr int kUnitBytes = kUnitGroups * 18 * kDim;
  static constexpr int kTileRows = MODE == kPairs ? 4 : 8;  // query rows of a tile
  static constexpr int kRows = NT * kTileRows;   // of a column group
  static constexpr int kSums = kStages * kWarps * kUnitBytes;                     // f32 [warp][row of a tile][d]
  static constexpr int kQuery = kSums + kWarps * kTileRows * kDim * 4;            // fp16 operand of the rows
  static constexpr int kQueryBytes = NT * NB * 512;                               // of a term
  static constexpr int kStats = kQuery + (MODE == kTwoTerms ? 2 : 1) * kQueryBytes;                     // f32 [warp][row][max, sum]
  static constexpr int kRowInfo = kStats + kWarps * kRows * 2 * 4;                // f32 scale, int position
  static constexpr int kFlags = kRowInfo + kRows * 8;                             // u32 [stage][warp]
  static constexpr int kBars = (kFlags + kStages * kWarps * 4 + 7) / 8 * 8;
  static constexpr int kBytes = kBars + kStages * kWarps * 8;
  static_assert(kBytes + 512 <= (NB * NT <= 4 ? 113 : 226) * 1024, "shared memory of an SM");
};

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same from zero.
__device__ __forceinline__ void mma16816_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// What lifts scales below `ceiling`, a power of two in 2^-24 .. 2^16, below 2^15: 2^15 / ceiling, exactly.
__device__ __forceinline__ float lift_of(float ceiling) {
  return __uint_as_float(((127u + 15u + 127u) << 23) - __float_as_uint(ceiling));
}

// 8 x 8 transpose of 16-bit elements held two to a lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) {
  uint32_t u;
  memcpy(&u, &h, 4);
  return u;
}
__device__ __forceinline__ __half2 bits_half2(uint32_t u) {
  __half2 h;
  memcpy(&h, &u, 4);
  return h;
}

// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t"
      ".reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\t"
      "mov.b64 b, {%4, %5};\n\t"
      "mov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\t"
      "mov.b64 {%0, %1}, d;\n\t"
      "}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t"
      ".reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\t"
      "mov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t"
      "}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t"
      ".reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\t"
      "mov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t"
      "}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Two nibbles n at bits 0..3 and 16..19 -> the fp16 pair n - 8: OR-ed into 1024.0 they are 1024 + n, and
// the subtraction is exact.  At bits 4..7 and 20..23 they make 1024 + 16 n: times 1/16, less 72.
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t u;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(u) : "r"(w), "r"(mask), "r"(bits));  // one instruction: (w & mask) | bits
  return u;
}
__device__ __forceinline__ uint32_t low_nibbles(uint32_t w) {
  const uint32_t u = and_or(w, 0x000f000fu, 0x64006400u);
  return half2_bits(__hsub2(bits_half2(u), bits_half2(0x64086408u)));
}
__device__ __forceinline__ uint32_t high_nibbles(uint32_t w) {
  const uint32_t u = and_or(w, 0x00f000f0u, 0x64006400u);
  return half2_bits(__hfma2(bits_half2(u), bits_half2(0x2c002c00u), bits_half2(0xd480d480u)));
}

// The words of one lane in one half of a group's quants, or one token's scales: N adjacent elements.
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t *p) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint2 v = reinterpret_cast<const uint2 *>(p)[i];
      w[2 * i] = v.x, w[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      w[i] = reinterpret_cast<const uint32_t *>(p)[i];
  }
}
// A token's NB scales, two to a word.
template <int NB>
__device__ __forceinline__ void load_scales(uint32_t (&w)[(NB + 1) / 2], const uint8_t *p) {
  if constexpr (NB % 2 == 0) {
    load_words<NB / 2>(w, p);
  } else {
#pragma unroll
    for (int i = 0; i < NB; i += 2)
      w[i / 2] = reinterpret_cast<const uint16_t *>(p)[i] | (i + 1 < NB ? static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(p)[i + 1]) << 16 : 0u);
  }
}
template <int N>
__device__ __forceinline__ float scale_of(const uint32_t (&w)[N], int b) {
  const __half2 h = bits_half2(w[b / 2]);
  return (b & 1) ? __high2float(h) : __low2float(h);
}

// What a call asks of one request.  `len` counts the tokens that its table has pages for; `before`, the position of its first row,
// goes by all the tokens and rows that the request has, also those that the table or the call leaves out.
struct Request {
  int32_t rows, first_row, len, before, first_unit, units, column_groups;
};

__device__ __forceinline__ Request load_request(const tcrv_cuda_attention_call &c, uint32_t group, uint32_t r, int group_rows) {
  Request q;
  long long first = c.first_rows ? c.first_rows[r] : r, end = c.first_rows ? c.first_rows[r + 1] : r + 1ll;
  if (first < 0)
    first = end = 0;
  const long long all = end - first;
  if (end > static_cast<long long>(c.rows))
    end = static_cast<long long>(c.rows);
  long long rows = end - first;
  rows = rows < 0 ? 0 : rows > static_cast<long long>(c.max_new) ? static_cast<long long>(c.max_new) : rows;
  const long long kv_len = c.kv_lens[r] < 0 ? 0 : c.kv_lens[r];
  const long long most = static_cast<long long>(c.width) * c.cache.groups * kGroupTokens;  // a whole number of groups
  const long long len = kv_len > most ? most : kv_len;
  q.rows = static_cast<int32_t>(rows);
  q.first_row = static_cast<int32_t>(first);
  q.len = static_cast<int32_t>(len);
  q.before = static_cast<int32_t>(kv_len - all);
  // the first row sees least far back
  long long low = c.window ? kv_len - all + 1 - static_cast<long long>(c.window) : 0;
  low = low < 0 ? 0 : low > len ? len : low;
  q.first_unit = static_cast<int32_t>(low / kUnitTokens);
  const int32_t units = static_cast<int32_t>((len + kUnitTokens - 1) / kUnitTokens) - q.first_unit;
  q.units = rows == 0 ? 0 : units < 1 ? 1 : units;  // (a request that sees nothing still writes its zeros)
  q.column_groups = static_cast<int32_t>((rows * group + group_rows - 1) / group_rows);
  return q;
}

// Positions are at most 2^31 - 2 and, held at -1 where a row sees nothing, at least -1: a window of 2^31 - 1 hides no token, and a
// position less a window fits 32 bits.
__device__ __forceinline__ int32_t window_of(const tcrv_cuda_attention_call &c) {
  return static_cast<int32_t>(c.window < 0x7fffffffu ? c.window : 0x7fffffffu);
}

// The same for the kernel of this file: requests with more rows than it is meant for have no units.
__device__ __forceinline__ Request load_request(const ColumnParams &p, uint32_t r, int group_rows) {
  Request q = load_request(p.call, p.group, r, group_rows);
  if (static_cast<long long>(q.rows) * p.group > p.most_rows)
    q.units = 0;
  return q;
}

__device__ __forceinline__ long long request_work(const ColumnParams &p, const Request &q) {
  return q.units == 0 ? 0 : static_cast<long long>(q.units + kSegmentUnits) * q.column_groups * static_cast<long long>(p.call.cache.kv_heads);
}

// A segment (kv head and column group of a request) of the list of all units: requests, then kv heads, then column groups,
// then units and behind them kSegmentUnits places without work.  Its ends count from the CTA's first place.
struct Cursor {
  uint32_t r;
  Request q;
  int32_t segment;  // head * column_groups + column group
  int32_t begin, end;
  // moves to the segment that holds unit u, which is not before this one (u is inside the list)
  __device__ __forceinline__ void seek(const ColumnParams &p, int32_t u, int group_rows) {
    while (u >= end) {
      begin = end;
      if (++segment == q.column_groups * static_cast<int32_t>(p.call.cache.kv_heads)) {
        segment = 0;
        do
          q = load_request(p, ++r, group_rows);
        while (q.units == 0);
      }
      end = begin + q.units + kSegmentUnits;
    }
  }
};

__device__ __forceinline__ long long cta_begin(long long work, int cta, int ctas) { return work * cta / ctas; }

// The list's length and the segment of this CTA's first unit.  Each thread sums a run of requests.
__device__ __forceinline__ long long find_start(const ColumnParams &p, int group_rows, long long *scratch, Cursor *out) {
  const uint32_t n = static_cast<uint32_t>(p.call.requests), per = (n + kThreads - 1) / kThreads;
  const uint32_t r0 = threadIdx.x * per, r1 = min(n, r0 + per);
  long long mine = 0;
  for (uint32_t r = r0; r < r1; ++r)
    mine += request_work(p, load_request(p, r, group_rows));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long s = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, s, off);
    if (lane >= off)
      s += o;
  }
  if (lane == 31)
    scratch[warp] = s;
  __syncthreads();
  long long before = s - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp)
      before += scratch[w];
    total += scratch[w];
  }
  const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), (total + kWarps - 1) / kWarps));
  if (static_cast<int>(blockIdx.x) < ctas) {
    const long long u = cta_begin(total, blockIdx.x, ctas);
    if (before <= u && u < before + mine) {
      Cursor c;
      for (c.r = r0;; ++c.r) {
        c.q = load_request(p, c.r, group_rows);
        const long long w = request_work(p, c.q);
        if (u < before + w)
          break;
        before += w;
      }
      const int32_t length = c.q.units + kSegmentUnits;
      c.segment = static_cast<int32_t>((u - before) / length);
      c.begin = static_cast<int32_t>(before + static_cast<long long>(c.segment) * length - u);
      c.end = c.begin + length;
      *out = c;
    }
  }
  __syncthreads();
  return total;
}

// One row's result: O / l, or zeros where nothing was seen; lse in natural units.
__device__ __forceinline__ void write_row(const tcrv_cuda_attention_call &c, size_t row, size_t head, uint32_t d, float sum,
                                          float l, float m) {
  store_typed(c.out, row * c.out_row_stride + head * c.out_head_stride + d, c.type, l > 0.0f || l != l ? sum / l : 0.0f);
  if (d == 0 && c.lse != nullptr)
    c.lse[row * c.heads + head] = l > 0.0f || l != l ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

// Work split: the list of all units (32 tokens of one kv head and column group) is cut into one range per
// CTA of equal length, whatever the contexts' lengths; inside a range the warps take units in turn, each
// with a ring of its own that its first two lanes fill by bulk copies ahead of use, across segment ends.  A
// segment that lies in one range is finished there; of one that does not, each CTA leaves maximum, sum and
// accumulators in the workspace for the combine kernel.
//
// Bound by instructions, not by the 9/16 byte a value: a warp's unit of D = 128 and 8 rows takes about 930 (32 words unpacked
// at 9 each, 32 products, the weights of each block, the soft-max, the scales' lift, the copies' addresses), issued in 60 % of the
// cycles by 16 warps.  2 x 131072 tokens, 32 / 8 heads, fp16: 93 us, 3.2 TB/s of cache; with (w & mask) | bits left to the compiler
// as two instructions, products that add to zeroed registers, and 64-bit cursors 200 instructions and a quarter more.  Rows of
// several tiles share a unit's unpacking (NT); their accumulators leave room for one CTA of 8 warps on an SM from 16 rows of 128 on,
// which covers no latencies: 16 x 5 drafted tokens, f32, 70 us with 30 % of the issue slots used.
template <int NB, int NT, int MODE>
__global__ void __launch_bounds__(kThreads, NB *NT <= 4 ? 2 : 1) columns_kernel(const __grid_constant__ ColumnParams p) {
  using L = ColumnLayout<NB, NT, MODE>;
  constexpr int kDim = L::kDim, kStages = L::kStages, kGroupBytes = 18 * kDim, kRows = L::kRows, kTileRows = L::kTileRows;
  constexpr int kMine = MODE == kPairs ? 1 : 2;  // query rows of a tile that a lane has
  const auto row_of = [](int t, int i) { return MODE == kPairs ? t : 2 * t + i; };
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long scratch[kWarps];
  __shared__ Cursor start;
  const tcrv_cuda_attention_call &c = p.call;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t *ring = smem + warp * kStages * L::kUnitBytes;
  float *sums = reinterpret_cast<float *>(smem + L::kSums);
  float *stats = reinterpret_cast<float *>(smem + L::kStats);
  float *row_scale = reinterpret_cast<float *>(smem + L::kRowInfo);
  int32_t *row_position = reinterpret_cast<int32_t *>(smem + L::kRowInfo) + kRows;
  volatile uint32_t *flags = reinterpret_cast<volatile uint32_t *>(smem + L::kFlags) + warp * kStages;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBars) + warp * kStages;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s)
      mbar_init(&bars[s], 1);
    mbar_fence_init();
  }
  pdl_enter();
  const long long work = find_start(p, kRows, scratch, &start);
  SplitRange *ranges = static_cast<SplitRange *>(c.workspace);
  const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), (work + kWarps - 1) / kWarps));
  if (static_cast<int>(blockIdx.x) >= ctas) {
    if (threadIdx.x == 0)
      ranges[blockIdx.x].valid = 0;
    return;
  }
  const long long u0 = cta_begin(work, blockIdx.x, ctas);
  const int32_t units = static_cast<int32_t>(cta_begin(work, blockIdx.x + 1, ctas) - u0);  // of this CTA, counted from 0

  // ---- this warp's copies: units warp, warp + kWarps, ...  Lanes 0 and 1 copy a group each; the page of the unit to
  // come is read one step before its copy, so that the copy never waits for the table.
  Cursor ahead = start;
  int32_t next = warp;  // unit whose pages are asked for
  const uint8_t *source = nullptr;
  const uint32_t per_page = static_cast<uint32_t>(c.cache.groups);
  const int page_shift = (per_page & (per_page - 1)) == 0 ? 31 - __clz(per_page) : -1;
  int32_t page = -1;
  size_t place = 0;
  auto fetch_page = [&]() {
    page = -1;
    for (;;) {  // (places without work are passed over, here and below)
      if (next >= units)
        return;
      ahead.seek(p, next, kRows);
      if (next - ahead.begin < ahead.q.units)
        break;
      next += (ahead.end - next + kWarps - 1) / kWarps * kWarps;
    }
    if (lane < kUnitGroups) {
      const uint32_t group = static_cast<uint32_t>(ahead.q.first_unit + (next - ahead.begin)) * kUnitGroups + lane;
      if (static_cast<int32_t>(group) * kGroupTokens < ahead.q.len) {
        const uint32_t at = page_shift >= 0 ? group >> page_shift : group / per_page;
        const uint32_t head = ahead.q.column_groups == 1 ? ahead.segment : ahead.segment / ahead.q.column_groups;
        page = c.block_table[ahead.r * c.table_stride + at];
        place = static_cast<size_t>(head * per_page + (group - at * per_page)) * kGroupBytes;
      }
    }
  };
  auto issue = [&](int stage) {
    if (next < units) {
      source = page >= 0 && static_cast<size_t>(page) < c.cache.pages ? c.cache.data + static_cast<size_t>(page) * c.cache.page_stride + place : nullptr;
      const uint32_t there = __ballot_sync(0xffffffffu, source != nullptr) & 3u;
      if (lane == 0) {
        flags[stage] = there;
        mbar_arrive_expect_tx(&bars[stage], __popc(there) * kGroupBytes);
      }
      __syncwarp();
      if (source != nullptr)
        bulk_copy_g2s(ring + stage * L::kUnitBytes + lane * kGroupBytes, source, kGroupBytes, &bars[stage]);
    }
    next += kWarps;
    fetch_page();
  };
  fetch_page();
#pragma unroll 1
  for (int s = 0; s < kStages; ++s)
    issue(s);
  int stage = 0;
  uint32_t parity = 0;
  bool failed = false;

  // The rows' operand: row i by warp i % kWarps.  The rows of the segment to come are read before the warps' parts of the
  // present one are joined, and placed meanwhile.
  float row_values[NT][NB];
  const auto load_rows = [&](const Cursor &of) {
    const int32_t head = of.segment / of.q.column_groups, pair0 = (of.segment - head * of.q.column_groups) * kRows;
    const int32_t pairs = min(kRows, of.q.rows * static_cast<int32_t>(p.group) - pair0);
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      const int i = k * kWarps + warp;
      const int32_t pair = pair0 + i, token = pair / static_cast<int32_t>(p.group);
      const int32_t q_head = head * static_cast<int32_t>(p.group) + (pair - token * static_cast<int32_t>(p.group));
#pragma unroll
      for (int b = 0; b < NB; ++b)
        row_values[k][b] = i < pairs ? load_typed(c.q, static_cast<size_t>(of.q.first_row + token) * c.q_row_stride +
                                                           static_cast<size_t>(q_head) * c.q_head_stride + b * 32 + lane, c.type)
                                     : 0.0f;
    }
  };
  const auto place_rows = [&](const Cursor &of) {
    const int32_t pair0 = (of.segment - of.segment / of.q.column_groups * of.q.column_groups) * kRows;
    const int32_t pairs = min(kRows, of.q.rows * static_cast<int32_t>(p.group) - pair0);
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      const int i = k * kWarps + warp;
      if (MODE == kPairs && i >= kRows)
        break;
      float top = 0.0f;
#pragma unroll
      for (int b = 0; b < NB; ++b)
        top = fmaxf(top, fabsf(row_values[k][b]));
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      // 2^power lifts the largest element into [2^14, 2^15); a row of zeros, or one with an infinity, stays
      const int power = top > 0.0f && top < INFINITY ? min(120, 141 - static_cast<int>(__float_as_uint(top) >> 23)) : 0;
      const float lift = __uint_as_float(static_cast<uint32_t>(127 + power) << 23);
      const int kstep = lane >> 4, f = lane & 15;
      __half *operand = reinterpret_cast<__half *>(smem + L::kQuery);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const float v = row_values[k][b] * lift;
        const __half hi = __float2half_rn(v);
        const int place = (((k * NB + b) * 32 + (MODE == kPairs ? 2 : 1) * warp * 4 + (f >> 2)) * 4 + kstep * 2 + (f & 1)) * 2 + ((f & 2) >> 1);
        operand[place] = hi;
        if constexpr (MODE != kOneTerm)  // (pairs: the column after it, four lanes on)
          operand[place + (MODE == kPairs ? 4 * 8 : L::kQueryBytes / 2)] = isfinite(v) ? __float2half_rn(v - __half2float(hi)) : __float2half_rn(0.0f);
      }
      if (lane == 0) {
        row_scale[i] = c.scale * kLog2e * __uint_as_float(static_cast<uint32_t>(127 - power) << 23);
        row_position[i] = i < pairs ? max(-1, of.q.before + (pair0 + i) / static_cast<int32_t>(p.group)) : -1;
      }
    }
  };

  Cursor at = start;
  int32_t u = warp;
  bool rows_here = false;
  if (threadIdx.x == 0)
    ranges[blockIdx.x].valid = 0;
  for (int32_t from = 0; from < units;) {
    at.seek(p, from, kRows);
    const int32_t seg_begin = at.begin, seg_end = at.begin + at.q.units, to = seg_end < units ? seg_end : units;
    if (seg_end <= from) {
      from = at.end;
      continue;
    }
    while (u < from)
      u += kWarps;
    const int32_t head = at.segment / at.q.column_groups, column_group = at.segment - head * at.q.column_groups;
    const int32_t pair0 = column_group * kRows, pairs = min(kRows, at.q.rows * static_cast<int32_t>(p.group) - pair0);

    if (!rows_here)
      load_rows(at);
    rows_here = true;
    place_rows(at);  // (no warp is still in the products of the segment before)
    __syncthreads();
    float scale[NT][kMine];
    int32_t position[NT][kMine];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int row = j * kTileRows + row_of(t, i);
        scale[j][i] = row_scale[row];
        position[j][i] = row_position[row];
      }
    // tokens that every row of the group sees (rows are in order of position)
    const int32_t window = window_of(c);
    const int32_t seen_to = row_position[0], seen_from = window ? row_position[pairs - 1] - window + 1 : 0;

    float m[NT][kMine], l[NT][kMine], o[2 * NB][NT][4];
    float ceiling = 0x1p-24f;  // the power of two above the largest value scale so far; the accumulators hold O * lift_of(ceiling)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < kMine; ++i)
        m[j][i] = -INFINITY, l[j][i] = 0.0f;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[i][j][e] = 0.0f;

    for (; u < to; u += kWarps) {
      if (!failed && !mbar_wait_bounded(&bars[stage], parity)) {
        failed = true;
        if (lane == 0)
          raise_device_error(p.errors, kDevErrBarrierTimeout);
        // no further copy; those on their way are waited for, with the same limit
        for (int s = 1; s < kStages && u + s * kWarps < units; ++s)
          mbar_wait_bounded(&bars[(stage + s) % kStages], parity ^ (stage + s >= kStages ? 1u : 0u));
        mbar_wait_bounded(&bars[stage], parity);
        next = units;
      }
      const uint8_t *unit = ring + stage * L::kUnitBytes;
      const uint32_t there = flags[stage];
      const int32_t token0 = (at.q.first_unit + (u - seg_begin)) * kUnitTokens;

      // ---- the largest value scale, a word or two to a lane (early, for the warp's maximum takes its time; NaN counts as nothing)
      __half2 most = __float2half2_rn(0.0f);
#pragma unroll
      for (int gr = 0; gr < kUnitGroups; ++gr)
#pragma unroll
        for (int i = 0; i < 8 * NB; i += 32)
          if (8 * NB % 32 == 0 || i + lane < 8 * NB)
            most = __hmax2(most, __habs2(*reinterpret_cast<const __half2 *>(unit + gr * kGroupBytes + 544 * NB + 4 * (i + lane))));
      uint32_t top_scale = __reduce_max_sync(0xffffffffu, __half_as_ushort(__hmax(__low2half(most), __high2half(most))));

      // ---- S^T = K q^T
      float s[kUnitGroups][NT][4];
#pragma unroll
      for (int gr = 0; gr < kUnitGroups; ++gr) {
        const uint8_t *group = unit + gr * kGroupBytes;
        uint32_t w0[NB], w1[NB];
        uint32_t d0[(NB + 1) / 2], d1[(NB + 1) / 2];
        load_words<NB>(w0, group + lane * NB * 4);
        load_words<NB>(w1, group + 128 * NB + lane * NB * 4);
        load_scales<NB>(d0, group + 512 * NB + g * NB * 2);
        load_scales<NB>(d1, group + 512 * NB + (g + 8) * NB * 2);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint32_t a0[4] = {low_nibbles(w0[b]), low_nibbles(w1[b]), low_nibbles(w0[b] >> 8), low_nibbles(w1[b] >> 8)};
          const uint32_t a1[4] = {high_nibbles(w0[b]), high_nibbles(w1[b]), high_nibbles(w0[b] >> 8), high_nibbles(w1[b] >> 8)};
          const float e[2] = {scale_of(d0, b), scale_of(d1, b)};
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint4 q = *reinterpret_cast<const uint4 *>(smem + L::kQuery + ((j * NB + b) * 32 + lane) * 16);
            float acc[4];
            mma16816_zero(acc, a0, q.x, q.y);
            mma16816(acc, a1, q.z, q.w);
            if constexpr (MODE == kTwoTerms) {
              const uint4 low = *reinterpret_cast<const uint4 *>(smem + L::kQuery + L::kQueryBytes + ((j * NB + b) * 32 + lane) * 16);
              mma16816(acc, a0, low.x, low.y);
              mma16816(acc, a1, low.z, low.w);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float2 x = make_float2(acc[2 * h], acc[2 * h + 1]), d = make_float2(e[h], e[h]);
              const float2 y = b == 0 ? mul2(x, d) : fma2(x, d, make_float2(s[gr][j][2 * h], s[gr][j][2 * h + 1]));
              s[gr][j][2 * h] = y.x;
              s[gr][j][2 * h + 1] = y.y;
            }
          }
        }
      }

      // ---- scores in powers of two, the mask, the running maximum and sum
      const bool whole = there == 3u && token0 >= seen_from && token0 + kUnitTokens - 1 <= seen_to;
      float pr[kUnitGroups][NT][2][kMine];  // [group][tile][token g or g + 8][row]
      bool moved = false;
      float alpha[NT][kMine];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          float top = -INFINITY;
#pragma unroll
          for (int gr = 0; gr < kUnitGroups; ++gr)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float v = (MODE == kPairs ? s[gr][j][2 * h] + s[gr][j][2 * h + 1] : s[gr][j][2 * h + i]) * scale[j][i];
              if (!whole) {
                const int32_t token = token0 + gr * kGroupTokens + h * 8 + g;
                if (!((there >> gr) & 1u) || token > position[j][i] || (window && token <= position[j][i] - window))
                  v = -INFINITY;
              }
              pr[gr][j][h][i] = v;
              top = fmaxf(top, v);
            }
#pragma unroll
          for (int off = 4; off <= 16; off <<= 1)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          const float now = fmaxf(m[j][i], top), base = now == -INFINITY ? 0.0f : now;
          alpha[j][i] = exp2_fast(m[j][i] - base);
          moved |= now != m[j][i];
          m[j][i] = now;
          float sum = 0.0f;
#pragma unroll
          for (int gr = 0; gr < kUnitGroups; ++gr)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              pr[gr][j][h][i] = exp2_fast(pr[gr][j][h][i] - base);
              sum += pr[gr][j][h][i];
            }
          l[j][i] = fmaf(l[j][i], alpha[j][i], sum);
        }

      // ---- value scales of this lane's tokens; those of tokens that no row sees may be anything and count as zero
      uint32_t vd[kUnitGroups][2][(NB + 1) / 2];
#pragma unroll
      for (int gr = 0; gr < kUnitGroups; ++gr)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          load_scales<NB>(vd[gr][h], unit + gr * kGroupBytes + 544 * NB + (g + 8 * h) * NB * 2);
          if (!whole) {
            const int32_t token = token0 + gr * kGroupTokens + h * 8 + g;
            const bool there_is = ((there >> gr) & 1u) && token <= row_position[pairs - 1] && !(window && token <= row_position[0] - window);
#pragma unroll
            for (int b = 0; b < (NB + 1) / 2; ++b)
              vd[gr][h][b] = there_is ? vd[gr][h][b] : 0u;
          }
        }
      // ---- the lift follows the largest of them that a row may see; beside infinities and NaNs it goes by the others
      if (!whole || top_scale >= 0x7c00u) {
        uint32_t top = 0;
#pragma unroll
        for (int gr = 0; gr < kUnitGroups; ++gr)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              const uint32_t d = (b & 1 ? vd[gr][h][b / 2] >> 16 : vd[gr][h][b / 2]) & 0x7fffu;
              top = max(top, d < 0x7c00u ? d : 0u);
            }
        top_scale = __reduce_max_sync(0xffffffffu, top);
      }
      const float top = half_bits_to_float(top_scale);
      float relift = 1.0f;
      if (top >= ceiling) {
        const uint32_t now = (__float_as_uint(top) & 0x7f800000u) + 0x00800000u;  // the next power of two
        relift = __uint_as_float(0x3f800000u + __float_as_uint(ceiling) - now);
        ceiling = __uint_as_float(now);
        moved = true;
      }
      const float lift = lift_of(ceiling);
#pragma unroll
      for (int gr = 0; gr < kUnitGroups; ++gr)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 x = mul2(make_float2(pr[gr][j][h][0], pr[gr][j][h][kMine - 1]), make_float2(lift, lift));
            pr[gr][j][h][0] = x.x;
            pr[gr][j][h][kMine - 1] = x.y;
          }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const float f0 = alpha[j][0] * relift, f1 = alpha[j][kMine - 1] * relift;
            o[i][j][0] *= f0;
            o[i][j][1] *= f1;
            o[i][j][2] *= f0;
            o[i][j][3] *= f1;
          }
      }

      // ---- O^T += V^T P^T, the weights times the value scales block by block
#pragma unroll
      for (int gr = 0; gr < kUnitGroups; ++gr) {
        const uint8_t *group = unit + gr * kGroupBytes + 256 * NB;
        uint32_t w0[NB], w1[NB];
        load_words<NB>(w0, group + lane * NB * 4);
        load_words<NB>(w1, group + 128 * NB + lane * NB * 4);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint32_t a0[4] = {low_nibbles(w0[b]), low_nibbles(w0[b] >> 8), low_nibbles(w1[b]), low_nibbles(w1[b] >> 8)};
          const uint32_t a1[4] = {high_nibbles(w0[b]), high_nibbles(w0[b] >> 8), high_nibbles(w1[b]), high_nibbles(w1[b] >> 8)};
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            constexpr int kProducts = MODE == kTwoTerms ? 2 : 1;
            uint32_t bits[kProducts][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float d = scale_of(vd[gr][h], b);
              if constexpr (MODE == kPairs) {
                float v = pr[gr][j][h][0] * d;
                if (!whole)
                  v = pr[gr][j][h][0] == 0.0f ? 0.0f : v;
                const float hi = __half2float(__float2half_rn(v));
                bits[0][h] = transpose8x8(half2_bits(__floats2half2_rn(hi, v - hi)));
              } else {
                float2 x = mul2(make_float2(pr[gr][j][h][0], pr[gr][j][h][kMine - 1]), make_float2(d, d));
                if (!whole) {  // a weight of zero stays zero, whatever the scale
                  x.x = pr[gr][j][h][0] == 0.0f ? 0.0f : x.x;
                  x.y = pr[gr][j][h][kMine - 1] == 0.0f ? 0.0f : x.y;
                }
                const __half2 hi = __floats2half2_rn(x.x, x.y);
                bits[0][h] = transpose8x8(half2_bits(hi));
                if constexpr (MODE == kTwoTerms) {
                  const float2 y = __half22float2(hi);
                  bits[kProducts - 1][h] = transpose8x8(half2_bits(__floats2half2_rn(x.x - y.x, x.y - y.y)));
                }
              }
            }
#pragma unroll
            for (int term = 0; term < kProducts; ++term) {
              mma16816(o[2 * b][j], a0, bits[term][0], bits[term][1]);
              mma16816(o[2 * b + 1][j], a1, bits[term][0], bits[term][1]);
            }
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      issue(stage);
      if (++stage == kStages) {
        stage = 0;
        parity ^= 1u;
      }
    }

    // ---- the warps' parts of the segment become one
    Cursor after = at;
    if (at.end < units) {
      after.seek(p, at.end, kRows);
      load_rows(after);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1)
          l[j][i] += __shfl_xor_sync(0xffffffffu, l[j][i], off);
        if (g == 0)
          stats[(warp * kRows + j * kTileRows + row_of(t, i)) * 2] = m[j][i];
      }
    __syncthreads();
    const bool first = seg_begin < 0, split = first || seg_end > units;
    const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (first ? 0 : 1);
    uint8_t *ws = static_cast<uint8_t *>(c.workspace);
    float *part_stats = reinterpret_cast<float *>(ws + column_stats_offset(gridDim.x)) + slot * kRows * 2;
    float *part_sums = reinterpret_cast<float *>(ws + column_sums_offset(gridDim.x, kRows)) + slot * kRows * kDim;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      // this warp's sums on the CTA's maximum
      float f[kMine];
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int row = j * kTileRows + row_of(t, i);
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
          top = fmaxf(top, stats[(w * kRows + row) * 2]);
        f[i] = m[j][i] == -INFINITY ? 0.0f : exp2_fast(m[j][i] - top);
        if (g == 0)
          stats[(warp * kRows + row) * 2 + 1] = l[j][i] * f[i];
        f[i] *= ceiling * 0x1p-15f;
      }
      float *mine = sums + warp * kTileRows * kDim;
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) {
        const int d = (i >> 1) * 32 + (i & 1) * 16 + 2 * g;
        if constexpr (MODE == kPairs) {
          *reinterpret_cast<float2 *>(mine + t * kDim + d) = make_float2((o[i][j][0] + o[i][j][1]) * f[0], (o[i][j][2] + o[i][j][3]) * f[0]);
        } else {
          *reinterpret_cast<float2 *>(mine + 2 * t * kDim + d) = make_float2(o[i][j][0] * f[0], o[i][j][2] * f[0]);
          *reinterpret_cast<float2 *>(mine + (2 * t + 1) * kDim + d) = make_float2(o[i][j][1] * f[kMine - 1], o[i][j][3] * f[kMine - 1]);
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < kTileRows * kDim; i += kThreads) {
        const int row = j * kTileRows + i / kDim, d = i % kDim;
        if (row >= pairs)
          break;
        float sum = 0.0f, total = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          sum += sums[w * kTileRows * kDim + i];
          total += stats[(w * kRows + row) * 2 + 1];
        }
        float top = 0.0f;
        if (d == 0) {
          top = -INFINITY;
#pragma unroll
          for (int w = 0; w < kWarps; ++w)
            top = fmaxf(top, stats[(w * kRows + row) * 2]);
        }
        if (split) {
          part_sums[row * kDim + d] = sum;
          if (d == 0) {
            part_stats[row * 2] = top;
            part_stats[row * 2 + 1] = total;
          }
        } else {
          const int32_t pair = pair0 + row, token = pair / static_cast<int32_t>(p.group);
          write_row(c, at.q.first_row + token, head * p.group + (pair - token * p.group), d, sum, total, top);
        }
      }
      if (j + 1 < NT)
        __syncthreads();
    }
    if (threadIdx.x == 0 && !first && seg_end > units) {  // the CTA that holds the segment's last unit
      const long long end = u0 + seg_end;
      int last = static_cast<int>((end - 1) * ctas / work);
      while (last + 1 < ctas && cta_begin(work, last + 1, ctas) < end)
        ++last;
      while (cta_begin(work, last, ctas) >= end)
        --last;
      SplitRange range = {};
      range.valid = 1;
      range.head = head;
      range.column_group = column_group;
      range.last_cta = last;
      range.rows = at.q.rows;
      range.first_row = at.q.first_row;
      ranges[blockIdx.x] = range;
    }
    from = at.end;
    at = after;
  }
}

// Joins the parts of a segment that several CTAs hold: block (c, y) does rows y, y + gridDim.y, ... of the segment
// that begins in CTA c and ends in a later one.
template <int NB>
__global__ void __launch_bounds__(kCombineThreads) columns_combine_kernel(const __grid_constant__ ColumnParams p, int rows) {
  constexpr int kDim = 32 * NB;
  __shared__ float reduce[2 * kCombineThreads / 32];
  pdl_enter();
  const tcrv_cuda_attention_call &c = p.call;
  const uint8_t *ws = static_cast<const uint8_t *>(c.workspace);
  const SplitRange range = static_cast<const SplitRange *>(c.workspace)[blockIdx.x];
  if (!range.valid)
    return;
  const float *stats = reinterpret_cast<const float *>(ws + column_stats_offset(gridDim.x));
  const float *sums = reinterpret_cast<const float *>(ws + column_sums_offset(gridDim.x, rows));
  const int32_t pair0 = range.column_group * rows, pairs = min(rows, range.rows * static_cast<int32_t>(p.group) - pair0);
  const int parts = range.last_cta - static_cast<int>(blockIdx.x) + 1;
  // part i: the second slot of the first CTA, the first slots of the others
  auto slot = [&](int i) { return 2 * static_cast<size_t>(blockIdx.x + i) + (i == 0 ? 1 : 0); };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int row = blockIdx.y; row < pairs; row += gridDim.y) {
    float top = -INFINITY;
    for (int i = threadIdx.x; i < parts; i += kCombineThreads)
      top = fmaxf(top, stats[(slot(i) * rows + row) * 2]);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1)
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if (lane == 0)
      reduce[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kCombineThreads / 32; ++w)
      top = fmaxf(top, reduce[w]);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum[(kDim + kCombineThreads - 1) / kCombineThreads] = {};
    float total = 0.0f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
      const float2 ml = *reinterpret_cast<const float2 *>(stats + (slot(i) * rows + row) * 2);
      const float f = exp2_fast(ml.x - base);
      total = fmaf(f, ml.y, total);
#pragma unroll
      for (int k = 0; k * kCombineThreads < kDim; ++k) {
        const int d = threadIdx.x + k * kCombineThreads;
        if (d < kDim)
          sum[k] = fmaf(f, sums[(slot(i) * rows + row) * kDim + d], sum[k]);
      }
    }
    const int32_t pair = pair0 + row, token = pair / static_cast<int32_t>(p.group);
#pragma unroll
    for (int k = 0; k * kCombineThreads < kDim; ++k) {
      const int d = threadIdx.x + k * kCombineThreads;
      if (d < kDim)
        write_row(c, range.first_row + token, range.head * p.group + (pair - token * p.group), d, sum[k], total, top);
    }
    __syncthreads();
  }
}

}  // namespace attention
}  // namespace tcrv
