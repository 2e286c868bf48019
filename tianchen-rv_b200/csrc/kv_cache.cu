// The paged Q4_0 key/value cache: a step's book-keeping (pages, slots, positions), the writer that
// quantises new rows into their slots, and the reader that gives slots back as numbers.
#include <cooperative_groups.h>

#include <atomic>

#include "kv_layout.cuh"
#include "launchers.h"

namespace tcrv {

namespace {

// ------------------------------------------------------------------ store and load

constexpr int kRowThreads = 256;
constexpr int kTeam = 4;  // lanes to a block of 32 elements: lane t has elements 4t..4t+3 and 16+4t..16+4t+3, so bytes 4t..4t+3

template <typename T>
__device__ __forceinline__ void load4(const T *p, bool vector, float *v) {
  if (vector) {
    if constexpr (sizeof(T) == 4) {
      const float4 x = *reinterpret_cast<const float4 *>(p);
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2 *>(p);
      T h[4];
      memcpy(h, &x, 8);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = to_float(h[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = to_float(p[i]);
  }
}

// Scale of a block and this lane's four bytes, by the rule of quantize_row_q4_0: the scale is the first element of largest
// magnitude over -8, a quant is trunc(x / d + 8.5), at most 15.  Every step is one IEEE operation or one that gives its bits
// (the product with -1/8, a power of two; the reciprocal), so the blocks are those of the row quantiser, byte for byte.
__device__ __forceinline__ uint32_t quantise_team(const float (&v)[8], float *scale) {
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    most = fmaxf(most, fabsf(v[j]));  // (NaN counts as nothing)
#pragma unroll
  for (int off = 1; off < kTeam; off <<= 1)
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
  // the first element of that magnitude: elements 0..15 lie across the lanes before 16..31 do
  float low = 0.0f, high = 0.0f;
  bool in_low = false, in_high = false;
#pragma unroll
  for (int j = 3; j >= 0; --j) {
    const bool l = fabsf(v[j]) == most, h = fabsf(v[4 + j]) == most;
    low = l ? v[j] : low;
    high = h ? v[4 + j] : high;
    in_low |= l;
    in_high |= h;
  }
  const int team = threadIdx.x & 28;
  const uint32_t holders_low = __ballot_sync(0xffffffffu, in_low) >> team & 15u, holders_high = __ballot_sync(0xffffffffu, in_high) >> team & 15u;
  const float chosen = __shfl_sync(0xffffffffu, holders_low ? low : high, __ffs(holders_low ? holders_low : holders_high) - 1, kTeam);
  const float best = most > 0.0f ? chosen : 0.0f;
  const float d = __fmul_rn(best, -0.125f);
  const float id = d != 0.0f ? __frcp_rn(d) : 0.0f;
  uint32_t bytes = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int q = static_cast<int>(__fadd_rn(__fmul_rn(v[j], id), 8.5f));  // (0 for NaN; far outside 0..15 where |d| < 2^-128, whose reciprocal is infinite)
    bytes |= static_cast<uint32_t>(max(0, min(15, q))) << (8 * (j & 3) + (j & 4));
  }
  *scale = d;
  return bytes;
}

// log2 of a power of two, -1 for other numbers
inline int shift_of(uint32_t n) {
  int s = 0;
  while (s < 31 && (1u << s) < n)
    ++s;
  return (1u << s) == n ? s : -1;
}

struct RowTensor {
  const void *p;
  size_t row_stride, head_stride;
};

// One team of four lanes per (row, head, block), the key's block and the value's; teams run over blocks, then heads, then
// rows, so a warp reads 8 adjacent blocks.  Bound by instructions, about 24 an element (8191 rows of 8 heads of 128, bf16:
// 35 us with eight lanes to a block, which pay the item's arithmetic and the shuffles twice); a key's words of one token are
// adjacent, a value's halfwords lie 4 bytes apart in 8 runs of 4 nb (they meet those of the group's other tokens in L2).
// kBlocks: blocks to a row, 0 where only the call knows.
template <typename T, bool kVector, int kBlocks>
__global__ void __launch_bounds__(kRowThreads)
    kv_store_kernel(RowTensor k, RowTensor v, const int64_t *slots, uint8_t *cache, size_t page_stride, int64_t capacity,
                    uint32_t page_tokens, int page_shift, Divisor by_row, Divisor by_block, uint32_t rows) {
  pdl_enter();
  const int t = threadIdx.x & (kTeam - 1);
  const uint32_t per_row = by_row.d, nb = kBlocks ? kBlocks : by_block.d;
  const uint64_t items = static_cast<uint64_t>(rows) * per_row;  // (fewer than 2^32)
  const uint64_t teams = static_cast<uint64_t>(gridDim.x) * (kRowThreads / kTeam);
  // (all teams of a warp make the same number of rounds: the shuffles need every lane)
  for (uint64_t first = static_cast<uint64_t>(blockIdx.x) * (kRowThreads / kTeam) + ((threadIdx.x >> 5) << 3); first < items; first += teams) {
    const uint64_t item = first + ((threadIdx.x & 31) / kTeam);
    const bool inside = item < items;
    const uint32_t row = inside ? by_row.of(static_cast<uint32_t>(item)) : 0;
    const uint32_t rest = inside ? static_cast<uint32_t>(item) - row * per_row : 0;
    const uint32_t head = kBlocks ? rest / nb : by_block.of(rest), b = rest - head * nb;
    const int64_t slot = inside ? slots[row] : -1;
    const bool live = slot >= 0 && slot < capacity;
    float kx[8], vx[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      kx[e] = vx[e] = 0.0f;
    if (live) {
      const T *kp = static_cast<const T *>(k.p) + row * k.row_stride + head * k.head_stride + b * 32 + 4 * t;
      const T *vp = static_cast<const T *>(v.p) + row * v.row_stride + head * v.head_stride + b * 32 + 4 * t;
      load4(kp, kVector, kx);
      load4(kp + 16, kVector, kx + 4);
      load4(vp, kVector, vx);
      load4(vp + 16, kVector, vx + 4);
    }
    float kd, vd;
    const uint32_t kq = quantise_team(kx, &kd), vq = quantise_team(vx, &vd);
    if (live) {
      const uint64_t page = page_shift >= 0 ? slot >> page_shift : static_cast<uint64_t>(slot) / page_tokens;
      const uint32_t in_page = static_cast<uint32_t>(slot - page * page_tokens), token = in_page % kGroupTokens;
      uint8_t *group = cache + page * page_stride +
                       static_cast<size_t>(head * (page_tokens / kGroupTokens) + in_page / kGroupTokens) * kv_group_bytes(32 * nb);
      *reinterpret_cast<uint32_t *>(group + kv_key_word(nb, token, t, b)) = kq;
      *reinterpret_cast<uint16_t *>(group + kv_value_half(nb, token, 2 * t, b)) = static_cast<uint16_t>(vq);
      *reinterpret_cast<uint16_t *>(group + kv_value_half(nb, token, 2 * t + 1, b)) = static_cast<uint16_t>(vq >> 16);
      if (t < 2)
        *reinterpret_cast<__half *>(group + (t == 0 ? kv_key_scale(nb, token, b) : kv_value_scale(nb, token, b))) = __float2half_rn(t == 0 ? kd : vd);
    }
  }
}

template <typename T>
__device__ __forceinline__ void store4(T *p, const float *v) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    T h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h[i] = from_float<T>(v[i]);
    uint2 x;
    memcpy(&x, h, 8);
    *reinterpret_cast<uint2 *>(p) = x;
  }
}

// The same items and lanes.  Bound by the bytes it writes.
template <typename T, int kBlocks>
__global__ void __launch_bounds__(kRowThreads)
    kv_load_kernel(T *k, T *v, const int64_t *slots, const uint8_t *cache, size_t page_stride, int64_t capacity,
                   uint32_t page_tokens, int page_shift, Divisor by_row, Divisor by_block, uint32_t rows) {
  pdl_enter();
  const int t = threadIdx.x & (kTeam - 1);
  const uint32_t per_row = by_row.d, nb = kBlocks ? kBlocks : by_block.d;
  const uint64_t items = static_cast<uint64_t>(rows) * per_row;  // (fewer than 2^32)
  const uint64_t teams = static_cast<uint64_t>(gridDim.x) * (kRowThreads / kTeam);
  for (uint64_t item = static_cast<uint64_t>(blockIdx.x) * (kRowThreads / kTeam) + threadIdx.x / kTeam; item < items; item += teams) {
    const uint32_t row = by_row.of(static_cast<uint32_t>(item)), rest = static_cast<uint32_t>(item) - row * per_row;
    const uint32_t head = kBlocks ? rest / nb : by_block.of(rest), b = rest - head * nb;
    const int64_t slot = slots[row];
    float kx[8], vx[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      kx[e] = vx[e] = 0.0f;
    if (slot >= 0 && slot < capacity) {
      const uint64_t page = page_shift >= 0 ? slot >> page_shift : static_cast<uint64_t>(slot) / page_tokens;
      const uint32_t in_page = static_cast<uint32_t>(slot - page * page_tokens), token = in_page % kGroupTokens;
      const uint8_t *group = cache + page * page_stride +
                             static_cast<size_t>(head * (page_tokens / kGroupTokens) + in_page / kGroupTokens) * kv_group_bytes(32 * nb);
      const uint32_t kq = *reinterpret_cast<const uint32_t *>(group + kv_key_word(nb, token, t, b));
      const uint32_t vq = *reinterpret_cast<const uint16_t *>(group + kv_value_half(nb, token, 2 * t, b)) |
                          static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(group + kv_value_half(nb, token, 2 * t + 1, b))) << 16;
      const float kd = __half2float(*reinterpret_cast<const __half *>(group + kv_key_scale(nb, token, b)));
      const float vd = __half2float(*reinterpret_cast<const __half *>(group + kv_value_scale(nb, token, b)));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = 8 * (e & 3) + (e & 4);
        kx[e] = __fmul_rn(kd, static_cast<float>(static_cast<int>((kq >> at) & 15u) - 8));
        vx[e] = __fmul_rn(vd, static_cast<float>(static_cast<int>((vq >> at) & 15u) - 8));
      }
    }
    const size_t at = static_cast<size_t>(item) * 32 + 4 * t;
    store4(k + at, kx);
    store4(k + at + 16, kx + 4);
    store4(v + at, vx);
    store4(v + at + 16, vx + 4);
  }
}

inline int row_grid(uint64_t items, int ctas_per_sm) {
  const uint64_t want = (items + kRowThreads / kTeam - 1) / (kRowThreads / kTeam);
  const uint64_t cap = static_cast<uint64_t>(sm_count()) * ctas_per_sm;
  return static_cast<int>(want < cap ? want : cap);
}

inline bool rows_aligned(const RowTensor &t, size_t element) {
  return reinterpret_cast<uintptr_t>(t.p) % (4 * element) == 0 && t.row_stride % 4 == 0 && t.head_stride % 4 == 0;
}

template <typename T>
int store_rows(const RowTensor &k, const RowTensor &v, size_t rows, const int64_t *slots, const tcrv_cuda_kv_cache &c,
               cudaStream_t stream) {
  const uint32_t nb = static_cast<uint32_t>(c.dim / 32), heads = static_cast<uint32_t>(c.kv_heads);
  const uint32_t page_tokens = static_cast<uint32_t>(c.groups * kGroupTokens);
  const int64_t capacity = static_cast<int64_t>(c.pages) * page_tokens;
  const int grid = row_grid(static_cast<uint64_t>(rows) * heads * nb, 8);
  const bool vector = rows_aligned(k, sizeof(T)) && rows_aligned(v, sizeof(T));
  auto *kernel = !vector ? kv_store_kernel<T, false, 0> : nb == 2 ? kv_store_kernel<T, true, 2> : nb == 4 ? kv_store_kernel<T, true, 4> : kv_store_kernel<T, true, 0>;
  TCRV_CUDA_TRY(launch_pdl(kernel, grid, kRowThreads, 0, stream, k, v, slots, c.data, c.page_stride, capacity, page_tokens,
                           shift_of(page_tokens), Divisor(heads * nb, static_cast<uint64_t>(rows) * heads * nb), Divisor(nb, heads * nb),
                           static_cast<uint32_t>(rows)));
  return TCRV_CUDA_OK;
}

template <typename T>
int load_rows(void *k, void *v, size_t rows, const int64_t *slots, const tcrv_cuda_kv_cache &c, cudaStream_t stream) {
  const uint32_t nb = static_cast<uint32_t>(c.dim / 32), heads = static_cast<uint32_t>(c.kv_heads);
  const uint32_t page_tokens = static_cast<uint32_t>(c.groups * kGroupTokens);
  const int64_t capacity = static_cast<int64_t>(c.pages) * page_tokens;
  const int grid = row_grid(static_cast<uint64_t>(rows) * heads * nb, 8);
  TCRV_CUDA_TRY(launch_pdl(nb == 2 ? kv_load_kernel<T, 2> : nb == 4 ? kv_load_kernel<T, 4> : kv_load_kernel<T, 0>, grid, kRowThreads, 0, stream, static_cast<T *>(k), static_cast<T *>(v), slots,
                           static_cast<const uint8_t *>(c.data), c.page_stride, capacity, page_tokens,
                           shift_of(page_tokens), Divisor(heads * nb, static_cast<uint64_t>(rows) * heads * nb), Divisor(nb, heads * nb),
                           static_cast<uint32_t>(rows)));
  return TCRV_CUDA_OK;
}

// ------------------------------------------------------------------ plan

constexpr int kPlanThreads = 1024;
constexpr int kPlanCtas = 8;           // one cluster of the portable size
// Rows and requests up to which one CTA does the step (device time, alone against a cluster: up to 8000 rows of 1000 requests the
// same 12 us, 4000 requests 20 against 16, 8000 requests 35 against 25).
constexpr uint32_t kPlanAlone = 2048;
constexpr size_t kPlanSmem = (3 * kPlanRequests + 2) * sizeof(int32_t);  // of the largest call

struct PlanSums {
  long long rows, pages;
};

// Exclusive sum of one value per thread over the CTA, and the total.
__device__ __forceinline__ PlanSums plan_scan(PlanSums v, PlanSums *warp_sums, PlanSums *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  PlanSums s = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long r = __shfl_up_sync(0xffffffffu, s.rows, off), p = __shfl_up_sync(0xffffffffu, s.pages, off);
    if (lane >= off) {
      s.rows += r;
      s.pages += p;
    }
  }
  if (lane == 31)
    warp_sums[warp] = s;
  __syncthreads();
  if (warp == 0) {
    PlanSums w = warp_sums[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long r = __shfl_up_sync(0xffffffffu, w.rows, off), p = __shfl_up_sync(0xffffffffu, w.pages, off);
      if (lane >= off) {
        w.rows += r;
        w.pages += p;
      }
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  *total = warp_sums[31];
  if (warp > 0) {
    s.rows += warp_sums[warp - 1].rows;
    s.pages += warp_sums[warp - 1].pages;
  }
  return {s.rows - v.rows, s.pages - v.pages};
}

// Index of the last of n ascending values that is <= x, given first[0] <= x.
__device__ __forceinline__ uint32_t plan_find(const int32_t *first, uint32_t n, int32_t x) {
  uint32_t low = 0, high = n;  // first[low] <= x < first[high]
  while (high - low > 1) {
    const uint32_t mid = (low + high) >> 1;
    if (first[mid] <= x)
      low = mid;
    else
      high = mid;
  }
  return low;
}

// Every CTA sums all requests (their two prefix sums stay in its shared memory), then the CTAs deal
// out the requests, the new pages and the rows among themselves; which request a page or row belongs
// to is found by bisection, so a step of one long prompt is as even as one of many tokens.  The cluster
// is there for inputs that outputs may replace (the free count, the lengths): nothing is written before all CTAs
// have read them.  Bound by latency: two dependent global reads, the scan, one write.
__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(tcrv_cuda_kv_plan_call c) {
  extern __shared__ int32_t plan_smem[];
  __shared__ PlanSums warp_sums[32];
  __shared__ int bad;
  const uint32_t n = static_cast<uint32_t>(c.requests), page = static_cast<uint32_t>(c.page_tokens);
  int32_t *first_row = plan_smem, *first_page = first_row + n + 1, *context = first_page + n + 1;
  if (threadIdx.x == 0)
    bad = 0;
  pdl_enter();
  __syncthreads();
  const long long free_count = *c.free_count;
  PlanSums base = {0, 0};
  int mine = 0;
  for (uint32_t r0 = 0; r0 < n; r0 += kPlanThreads) {
    const uint32_t r = r0 + threadIdx.x;
    PlanSums v = {0, 0};
    if (r < n) {
      const long long ctx = c.context_lens[r], add = c.new_lens[r];
      if (ctx < 0 || add < 0) {
        mine |= 2;
      } else {
        const long long need = (ctx + add + page - 1) / page;
        if (need > static_cast<long long>(c.width))
          mine |= 1;
        v = {add, need - (ctx + page - 1) / page};
      }
    }
    PlanSums total;
    const PlanSums at = plan_scan(v, warp_sums, &total);
    if (r < n) {  // (a sum beyond 31 bits is refused below)
      first_row[r] = static_cast<int32_t>(base.rows + at.rows);
      first_page[r] = static_cast<int32_t>(base.pages + at.pages);
      context[r] = c.context_lens[r];
    }
    base.rows += total.rows;
    base.pages += total.pages;
    __syncthreads();
  }
  if (mine)
    atomicOr(&bad, mine);
  if (threadIdx.x == 0) {
    first_row[n] = static_cast<int32_t>(base.rows);
    first_page[n] = static_cast<int32_t>(base.pages);
  }
  __syncthreads();
  int status = base.pages > free_count ? 1 : 0;
  if (bad & 1)
    status = 2;
  if (base.rows > static_cast<long long>(c.rows))
    status = 3;
  if ((bad & 2) || free_count < 0 || free_count > static_cast<long long>(c.free_capacity))
    status = 4;
  const bool ok = status == 0;

  if (gridDim.x > 1)
    cooperative_groups::this_cluster().sync();  // (kv_lens may be context_lens, info[3] the free count: all have read them)
  const uint32_t threads = gridDim.x * kPlanThreads, tid = blockIdx.x * kPlanThreads + threadIdx.x;
  for (uint32_t r = tid; r <= n; r += threads) {
    c.first_rows[r] = ok ? first_row[r] : 0;
    if (r < n)
      c.kv_lens[r] = ok ? context[r] + (first_row[r + 1] - first_row[r]) : context[r];
  }
  if (ok) {
    for (uint32_t j = tid; j < static_cast<uint32_t>(base.pages); j += threads) {
      const uint32_t r = plan_find(first_page, n, static_cast<int32_t>(j));
      const uint32_t held = (static_cast<uint32_t>(context[r]) + page - 1) / page;
      c.block_table[r * c.table_stride + held + (j - first_page[r])] = c.free_pages[free_count - 1 - j];
    }
  }
  const uint32_t used = ok ? static_cast<uint32_t>(base.rows) : 0;
  for (size_t i = tid; i < c.rows; i += threads) {
    int64_t slot = -1;
    int32_t position = 0, request = -1;
    if (i < used) {
      const uint32_t r = plan_find(first_row, n, static_cast<int32_t>(i));
      const uint32_t ctx = static_cast<uint32_t>(context[r]), held = (ctx + page - 1) / page;
      const uint32_t p = ctx + (static_cast<uint32_t>(i) - first_row[r]), at = p / page;
      const int32_t id = at < held ? c.block_table[r * c.table_stride + at]
                                   : c.free_pages[free_count - 1 - (first_page[r] + (at - held))];
      slot = static_cast<int64_t>(id) * page + (p - at * page);
      position = static_cast<int32_t>(p);
      request = static_cast<int32_t>(r);
    }
    c.slots[i] = slot;
    c.positions[i] = position;
    c.row_requests[i] = request;
  }
  if (tid == 0) {
    c.info[0] = status;
    c.info[1] = static_cast<int32_t>(used);
    c.info[2] = ok ? static_cast<int32_t>(base.pages) : 0;
    c.info[3] = static_cast<int32_t>(free_count - (ok ? base.pages : 0));
  }
}

}  // namespace

int launch_kv_store_q4_0(int type, size_t rows, const void *k, size_t k_row_stride, size_t k_head_stride, const void *v,
                         size_t v_row_stride, size_t v_head_stride, const int64_t *slots, const tcrv_cuda_kv_cache &cache,
                         cudaStream_t stream) {
  const RowTensor kt = {k, k_row_stride, k_head_stride}, vt = {v, v_row_stride, v_head_stride};
  if (type == TCRV_CUDA_TYPE_F32)
    return store_rows<float>(kt, vt, rows, slots, cache, stream);
  if (type == TCRV_CUDA_TYPE_F16)
    return store_rows<__half>(kt, vt, rows, slots, cache, stream);
  return store_rows<__nv_bfloat16>(kt, vt, rows, slots, cache, stream);
}

int launch_kv_load_q4_0(int type, size_t rows, void *k, void *v, const int64_t *slots, const tcrv_cuda_kv_cache &cache,
                        cudaStream_t stream) {
  if (type == TCRV_CUDA_TYPE_F32)
    return load_rows<float>(k, v, rows, slots, cache, stream);
  if (type == TCRV_CUDA_TYPE_F16)
    return load_rows<__half>(k, v, rows, slots, cache, stream);
  return load_rows<__nv_bfloat16>(k, v, rows, slots, cache, stream);
}

int launch_kv_plan(const tcrv_cuda_kv_plan_call &call, cudaStream_t stream) {
  const size_t smem = (3 * call.requests + 2) * sizeof(int32_t);
  // The limit without asking counts the kernel's static shared memory too, and an attribute is the process's: what the largest
  // call needs is asked for once on each device, before its first launch, and never taken back.
  static std::atomic<bool> done[64];
  int dev = 0;
  TCRV_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64)
    return TCRV_CUDA_ERR_UNSUPPORTED;
  if (!done[dev]) {
    TCRV_CUDA_TRY(cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kPlanSmem)));
    done[dev] = true;
  }
  const bool alone = call.requests <= kPlanAlone && call.rows <= kPlanAlone;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(alone ? 1 : kPlanCtas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = alone ? 1 : kPlanCtas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  TCRV_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv_plan_kernel, call));
  return TCRV_CUDA_OK;
}

}  // namespace tcrv
