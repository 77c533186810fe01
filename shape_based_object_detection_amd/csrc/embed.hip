// Rows of a label table, scaled, and the table's gradient by sorted labels.
//
//   out[i] = scale table[id_i];   d table[v] = scale sum over {i : id_i = v} of grad[i], in ascending i.
// An id outside [0, V) reads a row of zeros and gets no gradient; the padding id gets none.
//
// The gradient's order is fixed: the positions of each label are sorted first, one launch of workgroups
// that own a range of labels each, then each row of the table is summed by the threads that own its
// columns, in 32 bits, and written once (zeros where no label came): no atomics on sums, no clearing pass.
// A label that came often is summed in pieces first (k_embed_pieces), so that no thread walks a long run.
#include "label_dev.h"

namespace sbod {
namespace label {

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kSortRange = 512;    // labels per workgroup at most: 16 counts each, 32 KB of LDS
constexpr int kEmbThreads = 256;

// The table's row range a workgroup sorts: 256 workgroups where the vocabulary allows.
__host__ __device__ inline int64_t sort_range(int64_t v) {
  const int64_t r = (v + 255) / 256;
  return r < kSortRange ? r : kSortRange;
}

// Workgroup b: the positions of the labels [b range, (b + 1) range) in the order (label, position), and
// where each label's begin.  Every workgroup reads all ids (they stay in its XCD's L2): once to count
// its own labels and those below its range, once to place.  A wave owns a run of positions and a row of
// counters, so its placing needs no other wave: the order is that of the positions.
__global__ __launch_bounds__(kSortThreads) void k_embed_sort(const void *ids, int ids64, int64_t n, int64_t v,
                                                             int64_t padding, int range, int32_t *__restrict__ begin,
                                                             int32_t *__restrict__ sorted) {
  extern __shared__ int32_t cnt[];   // [kSortWaves][range]
  __shared__ int32_t red[kSortWaves], low[kSortWaves];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * range;
  const int mine = static_cast<int>(min(static_cast<int64_t>(range), v - lo));
  for (int i = threadIdx.x; i < kSortWaves * range; i += kSortThreads) cnt[i] = 0;
  __syncthreads();
  const int64_t per = ((n + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int64_t i0 = min(wv * per, n), i1 = min(i0 + per, n);
  int32_t *c = cnt + wv * range;
  int below = 0;
  constexpr int kU = 8;   // loads in flight per lane
  for (int64_t i = i0; i < i1; i += 64 * kU) {
    int id[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int64_t at = i + u * 64 + lane;
      id[u] = at < i1 ? ld_id(ids, at, ids64, v) : -1;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (id[u] < 0 || id[u] == padding) continue;
      if (id[u] < lo) ++below;
      else if (id[u] < lo + mine) atomicAdd(&c[id[u] - lo], 1);
    }
  }
  below = wave_sum_i32(below);
  if (lane == 0) low[wv] = below;
  __syncthreads();
  // thread t: label lo + t; the labels' exclusive sums over the workgroup, then each wave's start in each
  int tot = 0;
  if (static_cast<int>(threadIdx.x) < mine)
    for (int w = 0; w < kSortWaves; ++w) tot += cnt[w * range + threadIdx.x];
  int inc = tot;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(inc, d, kWave);
    if (lane >= d) inc += o;
  }
  if (lane == 63) red[wv] = inc;
  __syncthreads();
  int start = inc - tot;
  for (int w = 0; w < kSortWaves; ++w) {
    start += low[w];
    if (w < wv) start += red[w];
  }
  if (static_cast<int>(threadIdx.x) < mine) {
    begin[lo + threadIdx.x] = start;
    if (lo + threadIdx.x == v - 1) begin[v] = start + tot;
    int at = start;
    for (int w = 0; w < kSortWaves; ++w) {
      const int k = cnt[w * range + threadIdx.x];
      cnt[w * range + threadIdx.x] = at;
      at += k;
    }
  }
  __syncthreads();
  int bits = 0;
  while ((1 << bits) < mine) ++bits;
  volatile int32_t *place = c;
  for (int64_t i = i0; i < i1; i += 64 * kU) {
    int id[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int64_t at = i + u * 64 + lane;
      id[u] = at < i1 ? ld_id(ids, at, ids64, v) : -1;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const bool in = id[u] >= lo && id[u] < lo + mine && id[u] != padding;
      unsigned long long same = __ballot(in);
      if (same == 0) continue;
      const int key = in ? static_cast<int>(id[u] - lo) : 0;
      for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot(key >> b & 1);
        same &= key >> b & 1 ? set : ~set;
      }
      if (in) {
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const int at = place[key];
        sorted[at + rank] = static_cast<int32_t>(i + u * 64 + lane);
        wave_lds_fence();
        if (rank == 0) place[key] = at + __popcll(same);
      }
      wave_lds_fence();
    }
  }
}

// out[i] = scale table[id_i].  A block is rows x column groups of kV elements.
template <int DT, int kV>
__global__ __launch_bounds__(kEmbThreads) void k_embed_rows(const void *table, const void *ids, int ids64, int64_t n,
                                                            int64_t v, int64_t groups, float scale, void *out) {
  using T = typename Elt<DT>::T;
  using V = vec_t<T, kV>;
  const int64_t d = groups * kV;
  for (int64_t r = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y; r < n;
       r += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    const int id = ld_id(ids, r, ids64, v);
    const V *src = reinterpret_cast<const V *>(static_cast<const T *>(table) + (id < 0 ? 0 : id) * d);
    V *dst = reinterpret_cast<V *>(static_cast<T *>(out) + r * d);
    for (int64_t g = threadIdx.x; g < groups; g += blockDim.x) {
      V o;
      const V s = src[g];
#pragma unroll
      for (int j = 0; j < kV; ++j) o[j] = id < 0 ? static_cast<T>(0.f) : static_cast<T>(static_cast<float>(s[j]) * scale);
      dst[g] = o;
    }
  }
}

// Rows of a run per piece: about half the square root of the positions, so that a run's pieces are no
// more than the rows of one.
__host__ __device__ inline int piece_rows(int64_t n) {
  int s = 16;
  while (s < 1024 && 4ll * s * s < n) s *= 2;
  return s;
}

// acc += the rows sorted[b .. e) of grad, in that order; kU of them in flight.
template <typename T, int kV>
__device__ __forceinline__ void add_rows(float (&acc)[kV], const T *grad, const int32_t *sorted, int b, int e, int64_t d,
                                         int64_t g) {
  using V = vec_t<T, kV>;
  constexpr int kU = 8;
  for (int i = b; i < e; i += kU) {
    int at[kU];
    V s[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) at[u] = sorted[min(i + u, e - 1)];
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (i + u < e) s[u] = reinterpret_cast<const V *>(grad + at[u] * d)[g];
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (i + u < e) {
#pragma unroll
        for (int j = 0; j < kV; ++j) acc[j] += static_cast<float>(s[u][j]);
      }
  }
}

// Sums of the positions [c rows, (c + 1) rows) for the labels that came more than `rows` times: such a
// run covers the chunk's first position (pieces[c][0]) or, begun inside, its last one (pieces[c][1]).
template <int DT, int kV>
__global__ __launch_bounds__(kEmbThreads) void k_embed_pieces(const void *grad, const void *ids, int ids64,
                                                              const int32_t *begin, const int32_t *sorted, int64_t v,
                                                              int64_t chunks, int rows, int64_t groups, float *pieces) {
  using T = typename Elt<DT>::T;
  const int64_t d = groups * kV;
  const int total = begin[v];
  for (int64_t c = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y; c < chunks;
       c += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    const int c0 = static_cast<int>(c * rows), c1 = min(c0 + rows, total);
    if (c0 >= total) break;
    const int first = ld_id(ids, sorted[c0], ids64, v), last = ld_id(ids, sorted[c1 - 1], ids64, v);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int label = side ? last : first;
      if (side && last == first) break;
      const int b = begin[label], e = begin[label + 1];
      if (e - b <= rows) continue;
      for (int64_t g = threadIdx.x; g < groups; g += blockDim.x) {
        float acc[kV];
#pragma unroll
        for (int j = 0; j < kV; ++j) acc[j] = 0.f;
        add_rows<T, kV>(acc, static_cast<const T *>(grad), sorted, max(b, c0), min(e, c1), d, g);
        vec_t<float, kV> o;
#pragma unroll
        for (int j = 0; j < kV; ++j) o[j] = acc[j];
        reinterpret_cast<vec_t<float, kV> *>(pieces + (2 * c + side) * d)[g] = o;
      }
    }
  }
}

// d table[v] from the sorted positions.  The same blocks over the table's rows.
template <int DT, int kV>
__global__ __launch_bounds__(kEmbThreads) void k_embed_grad(const void *grad, const int32_t *begin,
                                                            const int32_t *sorted, int64_t v, int rows, int64_t groups,
                                                            const float *pieces, float scale, void *dtable) {
  using T = typename Elt<DT>::T;
  using V = vec_t<T, kV>;
  const int64_t d = groups * kV;
  for (int64_t r = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y; r < v;
       r += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    const int b = begin[r], e = begin[r + 1];
    V *dst = reinterpret_cast<V *>(static_cast<T *>(dtable) + r * d);
    for (int64_t g = threadIdx.x; g < groups; g += blockDim.x) {
      float acc[kV];
#pragma unroll
      for (int j = 0; j < kV; ++j) acc[j] = 0.f;
      if (e - b <= rows) {
        add_rows<T, kV>(acc, static_cast<const T *>(grad), sorted, b, e, d, g);
      } else {
        constexpr int kU = 4;
        const int last = (e - 1) / rows;
        for (int c = b / rows; c <= last; c += kU) {
          vec_t<float, kV> s[kU];
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            const int64_t at = min(c + u, last);
            s[u] = reinterpret_cast<const vec_t<float, kV> *>(pieces + (2 * at + (at * rows < b)) * d)[g];
          }
#pragma unroll
          for (int u = 0; u < kU; ++u)
            if (c + u <= last) {
#pragma unroll
              for (int j = 0; j < kV; ++j) acc[j] += s[u][j];
            }
        }
      }
      V o;
#pragma unroll
      for (int j = 0; j < kV; ++j) o[j] = static_cast<T>(acc[j] * scale);
      dst[g] = o;
    }
  }
}

// The widest column group that every row of both tensors starts on a multiple of.
int column_group(int64_t d, int dt, const void *p, const void *q) {
  const size_t b = elt_bytes(dt);
  int w = static_cast<int>(16 / b);
  while (w > 1 && (d % w != 0 || (reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) % (w * b) != 0)) w >>= 1;
  return w;
}

// kEmbThreads threads as (columns, rows): the columns a power of two that covers a row's groups.
dim3 row_block(int64_t groups) {
  int x = 1;
  while (x < kEmbThreads && x < groups) x <<= 1;
  return dim3(x, kEmbThreads / x);
}

dim3 row_grid(int64_t rows, dim3 block) {
  const int64_t b = (rows + block.y - 1) / block.y;
  return dim3(static_cast<unsigned>(b < 65536 ? b : 65536));
}

int check_embed(const char *what, int dt, int64_t n, int64_t v, int64_t d) {
  SBOD_REQUIRE(known_dt(dt), "%s: dtype %d", what, dt);
  SBOD_REQUIRE(n >= 0 && n < (1ll << 31) - 65536 && v >= 0 && v < (1ll << 31) - 65536 && d >= 0 && d < (1ll << 31),
               "%s: %lld labels, table [%lld, %lld]", what, static_cast<long long>(n), static_cast<long long>(v),
               static_cast<long long>(d));
  return SBOD_OK;
}

}  // namespace label
}  // namespace sbod

using namespace sbod;
using namespace sbod::label;

#define SBOD_EMBED_LAUNCH(KERNEL, DT, W, GRID, BLOCK, ...)                                            \
  do {                                                                                                \
    if ((DT) == SBOD_DT_F32) {                                                                        \
      if ((W) == 4) hipLaunchKernelGGL((KERNEL<SBOD_DT_F32, 4>), GRID, BLOCK, 0, s, __VA_ARGS__);      \
      else if ((W) == 2) hipLaunchKernelGGL((KERNEL<SBOD_DT_F32, 2>), GRID, BLOCK, 0, s, __VA_ARGS__); \
      else hipLaunchKernelGGL((KERNEL<SBOD_DT_F32, 1>), GRID, BLOCK, 0, s, __VA_ARGS__);               \
    } else if ((DT) == SBOD_DT_BF16) {                                                                \
      if ((W) == 8) hipLaunchKernelGGL((KERNEL<SBOD_DT_BF16, 8>), GRID, BLOCK, 0, s, __VA_ARGS__);     \
      else if ((W) == 4) hipLaunchKernelGGL((KERNEL<SBOD_DT_BF16, 4>), GRID, BLOCK, 0, s, __VA_ARGS__); \
      else if ((W) == 2) hipLaunchKernelGGL((KERNEL<SBOD_DT_BF16, 2>), GRID, BLOCK, 0, s, __VA_ARGS__); \
      else hipLaunchKernelGGL((KERNEL<SBOD_DT_BF16, 1>), GRID, BLOCK, 0, s, __VA_ARGS__);              \
    } else {                                                                                          \
      if ((W) == 8) hipLaunchKernelGGL((KERNEL<SBOD_DT_F16, 8>), GRID, BLOCK, 0, s, __VA_ARGS__);      \
      else if ((W) == 4) hipLaunchKernelGGL((KERNEL<SBOD_DT_F16, 4>), GRID, BLOCK, 0, s, __VA_ARGS__); \
      else if ((W) == 2) hipLaunchKernelGGL((KERNEL<SBOD_DT_F16, 2>), GRID, BLOCK, 0, s, __VA_ARGS__); \
      else hipLaunchKernelGGL((KERNEL<SBOD_DT_F16, 1>), GRID, BLOCK, 0, s, __VA_ARGS__);               \
    }                                                                                                 \
  } while (0)

extern "C" int sbod_embed_fwd(const void *table, int dtype, int64_t v, int64_t d, const void *ids, int ids64, int64_t n,
                              float scale, void *out, void *stream) {
  const int bad = check_embed("sbod_embed_fwd", dtype, n, v, d);
  if (bad != SBOD_OK) return bad;
  if (n == 0 || d == 0) return SBOD_OK;
  SBOD_REQUIRE(v > 0 && table && ids && out, "sbod_embed_fwd: empty table or null tensor");
  hipStream_t s = as_stream(stream);
  const int w = column_group(d, dtype, table, out);
  const dim3 block = row_block(d / w);
  SBOD_EMBED_LAUNCH(k_embed_rows, dtype, w, row_grid(n, block), block, table, ids, ids64, n, v, d / w, scale, out);
  SBOD_LAUNCHED("k_embed_rows");
  return SBOD_OK;
}

extern "C" size_t sbod_embed_bwd_workspace_bytes(int64_t n, int64_t v, int64_t d) {
  if (n < 0 || v <= 0 || d < 0) return 0;
  const int64_t rows = piece_rows(n), chunks = n > rows ? (n + rows - 1) / rows : 0;
  return align_up((v + 1) * sizeof(int32_t)) + align_up((n > 0 ? n : 1) * sizeof(int32_t)) +
         static_cast<size_t>(chunks) * 2 * d * sizeof(float);
}

extern "C" int sbod_embed_bwd(const void *grad, int dtype, int64_t v, int64_t d, const void *ids, int ids64, int64_t n,
                              int64_t padding, float scale, void *grad_table, void *workspace, size_t workspace_bytes,
                              void *stream) {
  const int bad = check_embed("sbod_embed_bwd", dtype, n, v, d);
  if (bad != SBOD_OK) return bad;
  if (v == 0 || d == 0) return SBOD_OK;
  SBOD_REQUIRE(grad_table && (n == 0 || (grad && ids)), "sbod_embed_bwd: null tensor");
  if (!workspace || workspace_bytes < sbod_embed_bwd_workspace_bytes(n, v, d)) {
    set_error("sbod_embed_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, sbod_embed_bwd_workspace_bytes(n, v, d));
    return SBOD_E_WORKSPACE;
  }
  hipStream_t s = as_stream(stream);
  int32_t *begin = static_cast<int32_t *>(workspace);
  int32_t *sorted = ws_at<int32_t>(workspace, align_up((v + 1) * sizeof(int32_t)));
  const int range = static_cast<int>(sort_range(v));
  hipLaunchKernelGGL(k_embed_sort, dim3(static_cast<unsigned>((v + range - 1) / range)), dim3(kSortThreads),
                     static_cast<size_t>(range) * kSortWaves * sizeof(int32_t), s, ids, ids64, n, v, padding, range, begin,
                     sorted);
  SBOD_LAUNCHED("k_embed_sort");
  const int w = column_group(d, dtype, grad, grad_table);
  const dim3 block = row_block(d / w);
  const int rows = piece_rows(n);
  float *pieces = nullptr;
  if (n > rows) {   // (else no label can have come more often)
    const int64_t chunks = (n + rows - 1) / rows;
    pieces = ws_at<float>(workspace, align_up((v + 1) * sizeof(int32_t)) + align_up(n * sizeof(int32_t)));
    SBOD_EMBED_LAUNCH(k_embed_pieces, dtype, w, row_grid(chunks, block), block, grad, ids, ids64, begin, sorted, v, chunks,
                      rows, d / w, pieces);
    SBOD_LAUNCHED("k_embed_pieces");
  }
  SBOD_EMBED_LAUNCH(k_embed_grad, dtype, w, row_grid(v, block), block, grad, begin, sorted, v, rows, d / w, pieces, scale,
                    grad_table);
  SBOD_LAUNCHED("k_embed_grad");
  return SBOD_OK;
}
