// Attention over the paged Q4_0 cache: choice of kernel, workspace, launches.
#include "attention_columns.cuh"
#include "launchers.h"

namespace tcrv {

namespace {

using namespace attention;

// Columns (query rows times their f32 terms) that one pass over a context takes, in tiles of 8: the fewest that hold
// all rows of a request, up to the tiles whose accumulators fit the registers.
int column_tiles(const tcrv_cuda_attention_call &c) {
  const int terms = c.type == TCRV_CUDA_TYPE_F32 ? 2 : 1;
  const size_t columns = c.max_new * (c.heads / c.cache.kv_heads) * terms;
  const int most = c.cache.dim <= 128 ? 4 : 2;
  for (int t = 1; t < most; t *= 2)
    if (columns <= static_cast<size_t>(8 * t))
      return t;
  return most;
}

struct Shape {
  int tiles, terms, rows;  // rows: query rows of a column group
  int grid;
};

Shape shape_of(const tcrv_cuda_attention_call &c) {
  Shape s;
  s.terms = c.type == TCRV_CUDA_TYPE_F32 ? 2 : 1;
  s.tiles = column_tiles(c);
  s.rows = s.tiles * 8 / s.terms;
  const size_t units = (c.width * c.cache.groups + kUnitGroups - 1) / kUnitGroups;
  const size_t groups = (c.max_new * (c.heads / c.cache.kv_heads) + s.rows - 1) / s.rows;
  const double most = static_cast<double>(units ? units : 1) * groups * c.cache.kv_heads * c.requests / kWarps + 1;
  const int cap = sm_count() * ctas_per_sm(static_cast<int>(c.cache.dim / 32), s.tiles);
  s.grid = most < cap ? static_cast<int>(most) : cap;
  return s;
}

template <int NB, int NT, int TERMS>
int launch_columns(const ColumnParams &p, const Shape &s, cudaStream_t stream) {
  constexpr size_t smem = ColumnLayout<NB, NT, TERMS>::kBytes;
  auto *kernel = columns_kernel<NB, NT, TERMS>;
  TCRV_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  TCRV_CUDA_TRY(launch_pdl(kernel, s.grid, kThreads, smem, stream, p));
  if (s.grid > 1) {
    const dim3 grid(static_cast<unsigned>(s.grid), static_cast<unsigned>(s.rows < 8 ? s.rows : 8));
    TCRV_CUDA_TRY(launch_pdl(columns_combine_kernel<NB>, grid, kCombineThreads, 0, stream, p, s.rows));
  }
  return TCRV_CUDA_OK;
}

template <int NB>
int launch_dim(const ColumnParams &p, const Shape &s, cudaStream_t stream) {
  if (s.terms == 1) {
    if (s.tiles == 1)
      return launch_columns<NB, 1, 1>(p, s, stream);
    if (s.tiles == 2)
      return launch_columns<NB, 2, 1>(p, s, stream);
    if constexpr (NB <= 4)
      return launch_columns<NB, 4, 1>(p, s, stream);
  } else {
    if (s.tiles == 1)
      return launch_columns<NB, 1, 2>(p, s, stream);
    if (s.tiles == 2)
      return launch_columns<NB, 2, 2>(p, s, stream);
    if constexpr (NB <= 4)
      return launch_columns<NB, 4, 2>(p, s, stream);
  }
  return TCRV_CUDA_ERR_UNSUPPORTED;
}

}  // namespace

size_t attention_workspace_bytes(const tcrv_cuda_attention_call &c) {
  const Shape s = shape_of(c);
  return column_workspace_bytes(s.grid, s.rows, c.cache.dim);
}

int launch_attention_q4_0(const tcrv_cuda_attention_call &c, cudaStream_t stream) {
  const Shape s = shape_of(c);
  ColumnParams p = {};
  p.call = c;
  p.group = static_cast<uint32_t>(c.heads / c.cache.kv_heads);
  const int st = device_error_words(&p.errors);
  if (st != TCRV_CUDA_OK)
    return st;
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
