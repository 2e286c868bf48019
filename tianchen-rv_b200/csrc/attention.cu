// Attention over the paged Q4_0 cache: choice of kernel, workspace, launches.
#include <atomic>

#include "attention_columns.cuh"
#include "attention_prefill.cuh"
#include "launchers.h"

namespace tcrv {

namespace {

using namespace attention;

// Rows of a request (new tokens * query heads of a kv head) from which its rows go to the prefill kernel, where there is one.  Contexts
// of 4096, 32 / 8 heads of 128, cold caches, columns kernel against prefill (bf16; bf16 with lse; fp16), us: 16 requests of 20 rows 83
// against 95 (bf16), of 32 rows 112 against 97, of 36 rows 140 against 93; 116; 126, of 64 rows 198 against the same; 64 requests of
// 20 rows 253 against 312, of 32 rows 372 against 314, of 36 rows 474 against 302; 392; 437; one request, whose few row blocks leave
// SMs idle, of 32 rows 26 against 41, of 64 rows 36 against 43; 45; 47, of 128 rows 46 against 45.
constexpr size_t kPrefillRows = 33;

struct Shape {
  // the columns kernel
  int tiles, mode, rows;  // rows: query rows of a column group, 8 to a tile (4 of kPairs)
  int grid;
  long long most_rows;
  // the prefill kernel
  bool prefill;
  int splits;
  size_t parts;
  size_t columns_bytes, prefill_offset, bytes;
};

Shape shape_of(const tcrv_cuda_attention_call &c) {
  Shape s = {};
  const size_t group = c.heads / c.cache.kv_heads, all = (c.max_new < c.rows ? c.max_new : c.rows) * group;
  s.prefill = all >= kPrefillRows && c.type != TCRV_CUDA_TYPE_F32 && (c.cache.dim == 64 || c.cache.dim == 128);
  const size_t rows = s.prefill ? kPrefillRows - 1 : all;
  s.most_rows = static_cast<long long>(rows);
  // the rows that one pass over a context takes, in tiles of 8: as many as have room for their sums in registers, dealt out evenly
  const size_t most_rows = 8 * (c.cache.dim <= 64 ? 4 : c.cache.dim <= 128 ? 3 : c.cache.dim <= 192 ? 2 : 1);
  const size_t groups = (rows + most_rows - 1) / most_rows;
  s.tiles = static_cast<int>(((rows + groups - 1) / groups + 7) / 8);
  s.mode = c.type != TCRV_CUDA_TYPE_F32 ? kOneTerm : rows <= 4 ? kPairs : kTwoTerms;
  s.rows = s.mode == kPairs ? 4 : 8 * s.tiles;
  const size_t units = (c.width * c.cache.groups + kUnitGroups - 1) / kUnitGroups;
  const double most = static_cast<double>((units ? units : 1) + kSegmentUnits) * groups * c.cache.kv_heads * c.requests / kWarps + 1;
  const int cap = sm_count() * ctas_per_sm(static_cast<int>(c.cache.dim / 32), s.tiles);
  s.grid = most < cap ? static_cast<int>(most) : cap;
  s.columns_bytes = column_workspace_bytes(s.grid, s.rows, c.cache.dim);
  s.prefill_offset = (s.columns_bytes + 255) / 256 * 256;
  s.bytes = s.columns_bytes;
  if (s.prefill) {
    const size_t items = (all + 2 * kTileRows - 1) / (2 * kTileRows) * c.requests * c.cache.kv_heads;
    // With fewer row blocks than half the SMs, each one's tokens are shared by several CTAs, of at least 4 tiles each (the last 64
    // tokens of 32768, whole and shared: 689 us, 80; the last 512 of 4096: 114, 81).  From half the SMs on the join costs more than
    // idle SMs (the last 1024 of 4096: 116, 154 shared).  At least one tile instead of 4: the last 64 of 4096 45 us instead of 54,
    // others the same or a little more; up to 148 parts instead of 32: 131072 tokens of one kv head 116 instead of 131, 32768 74
    // instead of 69.
    const size_t tiles = (c.width * c.cache.groups + kTileGroups - 1) / kTileGroups;
    size_t splits = items * 2 > static_cast<size_t>(sm_count()) ? 1 : sm_count() / items;
    splits = splits > (tiles + 3) / 4 ? (tiles + 3) / 4 : splits;
    s.splits = splits < 1 ? 1 : splits > 32 ? 32 : static_cast<int>(splits);
    s.parts = items * s.splits;
    if (s.splits > 1)
      s.bytes = s.prefill_offset + prefill_workspace_bytes(s.parts, c.cache.dim);
  }
  return s;
}

// What a kernel needs once on each device: its shared memory, and for one that splits its registers the proof that a block
// starts with as many (a block with fewer would wait for them for ever).
struct Configured {
  std::atomic<bool> done[64];
};
int configure(Configured &state, const void *kernel, size_t smem, int threads, int registers) {
  int dev = 0;
  TCRV_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64)
    return TCRV_CUDA_ERR_UNSUPPORTED;
  if (!state.done[dev]) {
    cudaFuncAttributes attributes;
    TCRV_CUDA_TRY(cudaFuncGetAttributes(&attributes, kernel));
    if (attributes.numRegs * threads < registers)
      return TCRV_CUDA_ERR_UNSUPPORTED;
    TCRV_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    state.done[dev] = true;
  }
  return TCRV_CUDA_OK;
}

template <int NB, int NT, int MODE>
int launch_columns(const ColumnParams &p, const Shape &s, cudaStream_t stream) {
  constexpr size_t smem = ColumnLayout<NB, NT, MODE>::kBytes;
  auto *kernel = columns_kernel<NB, NT, MODE>;
  static Configured state;
  const int st = configure(state, reinterpret_cast<const void *>(kernel), smem, kThreads, 0);
  if (st != TCRV_CUDA_OK)
    return st;
  TCRV_CUDA_TRY(launch_pdl(kernel, s.grid, kThreads, smem, stream, p));
  if (s.grid > 1) {
    const dim3 grid(static_cast<unsigned>(s.grid), static_cast<unsigned>(s.rows < 8 ? s.rows : 8));
    TCRV_CUDA_TRY(launch_pdl(columns_combine_kernel<NB>, grid, kCombineThreads, 0, stream, p, s.rows));
  }
  return TCRV_CUDA_OK;
}

template <int NB, int MODE>
int launch_tiles(const ColumnParams &p, const Shape &s, cudaStream_t stream) {
  switch (s.tiles) {
    case 1:
      return launch_columns<NB, 1, MODE>(p, s, stream);
    case 2:
      if constexpr (NB <= 6)
        return launch_columns<NB, 2, MODE>(p, s, stream);
      break;
    case 3:
      if constexpr (NB <= 4)
        return launch_columns<NB, 3, MODE>(p, s, stream);
      break;
    case 4:
      if constexpr (NB <= 2)
        return launch_columns<NB, 4, MODE>(p, s, stream);
      break;
  }
  return TCRV_CUDA_ERR_UNSUPPORTED;
}

template <int NB>
int launch_dim(const ColumnParams &p, const Shape &s, cudaStream_t stream) {
  return s.mode == kOneTerm ? launch_tiles<NB, kOneTerm>(p, s, stream)
         : s.mode == kPairs ? launch_columns<NB, 1, kPairs>(p, s, stream)
                            : launch_tiles<NB, kTwoTerms>(p, s, stream);
}

template <int NB, int MODE>
int launch_prefill(const tcrv_cuda_attention_call &c, const Shape &s, const DeviceErrorWords &errors, cudaStream_t stream) {
  if (s.parts > 0x7fffffff)
    return TCRV_CUDA_ERR_UNSUPPORTED;
  PrefillParams p = {};
  p.call = c;
  p.call.workspace = static_cast<uint8_t *>(c.workspace) + s.prefill_offset;
  p.group = static_cast<uint32_t>(c.heads / c.cache.kv_heads);
  p.min_rows = static_cast<int32_t>(kPrefillRows);
  p.splits = s.splits;
  p.errors = errors;
  constexpr size_t smem = PrefillLayout<NB, MODE>::kBytes;
  static Configured state;
  const int st = configure(state, reinterpret_cast<const void *>(prefill_kernel<NB, MODE>), smem, kPrefillThreads,
                           128 * (2 * kSoftmaxRegs + 2 * kQuantRegs + kProductRegs));
  if (st != TCRV_CUDA_OK)
    return st;
  TCRV_CUDA_TRY(launch_pdl(prefill_kernel<NB, MODE>, dim3(static_cast<unsigned>(s.parts)), kPrefillThreads, smem, stream, p));
  if (s.splits > 1) {
    const dim3 grid(2 * kTileRows / 8, static_cast<unsigned>(s.parts / s.splits));
    TCRV_CUDA_TRY(launch_pdl(prefill_combine_kernel<NB>, grid, 256, 0, stream, p, static_cast<uint32_t>(s.parts)));
  }
  return TCRV_CUDA_OK;
}

}  // namespace

size_t attention_workspace_bytes(const tcrv_cuda_attention_call &c) { return shape_of(c).bytes; }

int launch_attention_q4_0(const tcrv_cuda_attention_call &c, cudaStream_t stream) {
  const Shape s = shape_of(c);
  ColumnParams p = {};
  p.call = c;
  p.group = static_cast<uint32_t>(c.heads / c.cache.kv_heads);
  p.most_rows = s.most_rows;
  const int st = device_error_words(&p.errors);
  if (st != TCRV_CUDA_OK)
    return st;
  if (s.prefill) {
    // as exact as the outputs show: fp16 results both roundings, an f32 lse that of the keys, bf16 results neither
    const auto launch = [&](auto dim) {
      constexpr int kBlocks = decltype(dim)::value;
      return c.type == TCRV_CUDA_TYPE_F16 ? launch_prefill<kBlocks, kExactAll>(c, s, p.errors, stream)
             : c.lse != nullptr           ? launch_prefill<kBlocks, kExactKeys>(c, s, p.errors, stream)
                                          : launch_prefill<kBlocks, kRounded>(c, s, p.errors, stream);
    };
    const int rc = c.cache.dim == 64 ? launch(std::integral_constant<int, 2>()) : launch(std::integral_constant<int, 4>());
    if (rc != TCRV_CUDA_OK)
      return rc;
  }
  switch (c.cache.dim) {
    case 64:
      return launch_dim<2>(p, s, stream);
    case 96:
      return launch_dim<3>(p, s, stream);
    case 128:
      return launch_dim<4>(p, s, stream);
    case 192:
      return launch_dim<6>(p, s, stream);
    case 256:
      return launch_dim<8>(p, s, stream);
    default:
      return TCRV_CUDA_ERR_UNSUPPORTED;
  }
}

}  // namespace tcrv
