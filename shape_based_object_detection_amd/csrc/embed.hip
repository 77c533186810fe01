// Rows of a label table, scaled, and the table's gradient by sorted labels.
//
//   out[i] = scale table[id_i];   d table[v] = scale sum over {i : id_i = v} of grad[i].
// An id outside [0, V) reads a row of zeros and gets no gradient; the padding id gets none.
//
// The gradient's order is fixed by the call's ids and sizes: the positions of each label are sorted first, one launch of workgroups
// that own a range of labels each, then each row of the table is summed by the threads that own its
// columns, in 32 bits, and written once (zeros where no label came): no atomics on sums, no clearing pass.
// A label that came often is summed in pieces first (k_embed_pieces), so that no thread walks a long run: in
// ascending position within a piece, the pieces in that order; where they are cut depends on how many labels
// below it the call has.
// Few labels at few positions take one launch instead (k_embed_few).
#include <type_traits>

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

// Positions per flag bit of a wave's run of `per` positions: 64, or more so that a wave's flags fit
// kSortFlags words (64 positions up to 4 M ids).
constexpr int kSortFlags = 64;
__host__ __device__ inline int flag_shift(int64_t per) {
  int shift = 6;
  while (per > (64ll * kSortFlags) << shift) ++shift;
  return shift;
}

// Workgroup b: the positions of the labels [b range, (b + 1) range) in the order (label, position), and
// where each label's begin (an absent id has no place).  Every workgroup reads all ids (they stay in its
// XCD's L2), counts its own labels and those below its range, and flags the stretches that hold one of
// its own: only those are read again, to place.  A wave owns a run of positions and a row of counters, so
// its placing needs no other wave: the order is that of the positions.  Bound by the latency of its passes: 54 us
// for 65,536 ids of 131,072 labels, 11 for 8,192 of 32,000; its reads grow as ids times labels above 131,072 labels.
template <typename ID>
__global__ __launch_bounds__(kSortThreads) void k_embed_sort(const ID *__restrict__ ids, int64_t n, int64_t v, int range,
                                                             int32_t *__restrict__ begin, int32_t *__restrict__ sorted) {
  using U = std::make_unsigned_t<ID>;   // (a negative id is above every label)
  extern __shared__ int32_t cnt[];      // [kSortWaves][range]
  __shared__ int32_t red[kSortWaves], low[kSortWaves];
  __shared__ unsigned long long flags[kSortWaves][kSortFlags];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const U lo = static_cast<U>(static_cast<int64_t>(blockIdx.x) * range);
  const int mine = static_cast<int>(min(static_cast<int64_t>(range), v - static_cast<int64_t>(lo)));
  for (int i = threadIdx.x; i < kSortWaves * range; i += kSortThreads) cnt[i] = 0;
  flags[wv][lane] = 0;
  __syncthreads();
  const int64_t per = ((n + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int shift = flag_shift(per);
  const int64_t i0 = min(wv * per, n), i1 = min(i0 + per, n);
  int32_t *c = cnt + wv * range;
  int below = 0;
  constexpr int kU = 8;   // loads in flight per lane
  for (int64_t i = i0; i < i1; i += 64 * kU) {
    U id[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int64_t at = i + u * 64 + lane;
      id[u] = at < i1 ? static_cast<U>(ids[at]) : ~static_cast<U>(0);
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      below += __popcll(__ballot(id[u] < lo));
      const U at = id[u] - lo;
      const bool in = at < static_cast<U>(mine);
      if (__ballot(in) == 0) continue;
      if (in) atomicAdd(&c[static_cast<int>(at)], 1);
      const int64_t f = (i + u * 64 - i0) >> shift;
      if (lane == 0) flags[wv][f >> 6] |= 1ull << (f & 63);
    }
  }
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
    const int64_t label = static_cast<int64_t>(lo) + threadIdx.x;
    begin[label] = start;
    if (label == v - 1) begin[v] = start + tot;
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
  const int words = static_cast<int>((i1 - i0 + (64ll << shift) - 1) >> (shift + 6));   // of flags in use
  for (int word = 0; word < words; ++word) {
    // (read into scalar registers: the walk below is the same for every lane)
    unsigned long long left = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(flags[wv][word] >> 32)));
    left = left << 32 | static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(flags[wv][word])));
    int64_t stretch = 0, end = 0;   // of a longer stretch: what is left of it
    while (left || stretch < end) {
      // the next kU groups of 64 positions, in order: their loads overlap
      int64_t from[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (stretch >= end && left) {
          stretch = i0 + ((static_cast<int64_t>(word) * 64 + __ffsll(left) - 1) << shift);
          end = stretch + (1ll << shift);
          left &= left - 1;
        }
        from[u] = stretch < end ? stretch : i1;
        if (stretch < end) stretch += 64;
      }
      U id[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int64_t at = from[u] + lane;
        id[u] = at < i1 ? static_cast<U>(ids[at]) : ~static_cast<U>(0);
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const U at = id[u] - lo;
        const bool in = at < static_cast<U>(mine);
        unsigned long long todo = __ballot(in);
        const int key = in ? static_cast<int>(at) : -1;
        const int32_t pos = static_cast<int32_t>(from[u] + lane);
        const unsigned long long before = (1ull << lane) - 1;
        if (__popcll(todo) <= 16) {   // few of this workgroup's: label by label
          while (todo) {
            const int k0 = __builtin_amdgcn_readlane(key, __ffsll(todo) - 1);
            const unsigned long long same = __ballot(key == k0);
            const int first = place[k0];
            if (key == k0) sorted[first + __popcll(same & before)] = pos;
            wave_lds_fence();
            if (lane == 0) place[k0] = first + __popcll(same);
            wave_lds_fence();
            todo &= ~same;
          }
        } else {   // many: the lanes of the same label by the bits of it
          unsigned long long same = todo;
          for (int b = 0; b < bits; ++b) {
            const unsigned long long set = __ballot(key >> b & 1);
            same &= key >> b & 1 ? set : ~set;
          }
          if (in) {
            const int rank = __popcll(same & before);
            const int first = place[key];
            sorted[first + rank] = pos;
            wave_lds_fence();
            if (rank == 0) place[key] = first + __popcll(same);
          }
          wave_lds_fence();
        }
      }
    }
  }
}

// out[i] = scale table[id_i].  A block is rows x column groups of kV elements.  Bound by memory: 143 us for 65,536
// rows of 4,096 bfloat16 elements (537 MB written and the rows read: 5.2 TB/s), 3 us for 32 of them.
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

// Rows of a run per piece: about a quarter of the square root of the positions, 16 at least and 1024 at
// most, so that neither a piece's rows nor a run's pieces are many.
__host__ __device__ inline int piece_rows(int64_t n) {
  int s = 16;
  while (s < 1024 && 16ll * s * s < n) s *= 2;
  return s;
}

// acc += the rows sorted[b .. e) of grad, in that order; kU of them in flight, and the next ones' numbers.
template <typename T, int kV>
__device__ __forceinline__ void add_rows(float (&acc)[kV], const T *grad, const int32_t *sorted, int b, int e, int64_t d,
                                         int64_t g) {
  using V = vec_t<T, kV>;
  constexpr int kU = 8;
  if (b >= e) return;
  int at[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) at[u] = sorted[min(b + u, e - 1)];
  int i = b;
  for (; i + kU <= e; i += kU) {   // whole batches: loads without a branch between them
    V s[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) s[u] = reinterpret_cast<const V *>(grad + at[u] * d)[g];
#pragma unroll
    for (int u = 0; u < kU; ++u) at[u] = sorted[min(i + kU + u, e - 1)];
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int j = 0; j < kV; ++j) acc[j] += static_cast<float>(s[u][j]);
  }
  if (i < e) {
    V s[kU];
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
// run covers the chunk's first position (pieces[c][0]) or, begun inside, its last one (pieces[c][1]).  Bound by
// its reads: 76 us where 65,536 positions follow their labels' frequencies (1 / rank), 4,096 columns.
template <int DT, int kV>
__global__ __launch_bounds__(kEmbThreads) void k_embed_pieces(const void *grad, const void *ids, int ids64,
                                                              const int32_t *begin, const int32_t *sorted, int64_t v,
                                                              int64_t padding, int64_t chunks, int rows, int64_t groups,
                                                              float *pieces) {
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
      if (e - b <= rows || label == padding) continue;
      const int64_t g = blockIdx.y * static_cast<int64_t>(blockDim.x) + threadIdx.x;
      if (g < groups) {
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

// d table[v] from the sorted positions.  The same blocks over the table's rows, kEmbRows of them per thread:
// most labels came once or not at all, so a row is a chain of three loads (its places, their first row's
// number, that row), and the rows' chains run side by side: 305 us for 65,536 positions into
// a table of 1 GB (before its stores went past the caches 395 with 4 rows, 453 with 1).
template <int DT, int kV, int kEmbRows>
__global__ __launch_bounds__(kEmbThreads) void k_embed_grad(const void *grad, const int32_t *begin,
                                                            const int32_t *sorted, int64_t v, int64_t padding, int rows,
                                                            int64_t groups, const float *pieces, float scale,
                                                            void *dtable) {
  using T = typename Elt<DT>::T;
  using V = vec_t<T, kV>;
  const int64_t d = groups * kV;
  const int64_t g = blockIdx.y * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  if (g >= groups) return;
  const T *src = static_cast<const T *>(grad);
  for (int64_t r0 = (blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y) * kEmbRows; r0 < v;
       r0 += static_cast<int64_t>(gridDim.x) * blockDim.y * kEmbRows) {
    int at[kEmbRows + 1], first[kEmbRows];
    V one[kEmbRows];
#pragma unroll
    for (int k = 0; k <= kEmbRows; ++k) at[k] = begin[min(r0 + k, v)];
#pragma unroll
    for (int k = 0; k < kEmbRows; ++k) first[k] = at[k] < at[k + 1] ? sorted[at[k]] : -1;
#pragma unroll
    for (int k = 0; k < kEmbRows; ++k)
      if (first[k] >= 0) one[k] = reinterpret_cast<const V *>(src + first[k] * d)[g];
#pragma unroll
    for (int k = 0; k < kEmbRows; ++k) {
      const int64_t r = r0 + k;
      if (r >= v) break;
      const int b = at[k], e = r == padding ? b : at[k + 1];
      float acc[kV];
#pragma unroll
      for (int j = 0; j < kV; ++j) acc[j] = 0.f;
      if (e - b <= rows) {
        if (b < e) {
#pragma unroll
          for (int j = 0; j < kV; ++j) acc[j] = static_cast<float>(one[k][j]);
          add_rows<T, kV>(acc, src, sorted, b + 1, e, d, g);
        }
      } else {
        constexpr int kU = 4;
        const int last = (e - 1) / rows;
        for (int c = b / rows; c <= last; c += kU) {
          vec_t<float, kV> s[kU];
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            const int64_t p = min(c + u, last);
            s[u] = reinterpret_cast<const vec_t<float, kV> *>(pieces + (2 * p + (p * rows < b)) * d)[g];
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
      // (written once and not read here: past the caches: the backward pass of a 1 GB table 505 against 535 us)
      __builtin_nontemporal_store(o, reinterpret_cast<V *>(static_cast<T *>(dtable) + r * d) + g);
    }
  }
}

// d table of few labels from few positions, in one launch and without a sort.  A workgroup has a label and a tile
// of columns: its waves look through 512 positions each for the label's and list them in order, its threads, as
// (columns, slots), add every slots'th row of the list, and the slots are joined: in a wave by lane swaps, the waves'
// sums in LDS.  Bound by the latency of that chain: 7 us for 6,400 positions of 21 labels, 256 float32 columns (the
// sort and what is behind it 18 in three launches), 21 where all 8,192 have one label (49).
constexpr int kFewWave = 512;              // positions of a wave
constexpr int kFewMost = 16 * kFewWave;    // of a workgroup of 1,024 threads
constexpr int kFewCols = 64;               // columns of a tile
template <int DT, int kV>
__global__ __launch_bounds__(1024) void k_embed_few(const void *grad, const void *ids, int ids64, int n, int64_t v,
                                                    int64_t padding, int64_t groups, int lanes, float scale, void *dtable) {
  using T = typename Elt<DT>::T;
  using V = vec_t<T, kV>;
  constexpr int kSteps = kFewWave / kWave;
  __shared__ uint16_t list[kFewMost];
  __shared__ int counts[16];
  __shared__ float part[16][kFewCols];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, waves = blockDim.x >> 6, label = blockIdx.x;
  const int first = wv * kFewWave + lane;
  RawId raw[kSteps];
#pragma unroll
  for (int u = 0; u < kSteps; ++u) raw[u] = ld_raw_id(ids, min(first + u * kWave, n - 1), ids64);
  unsigned long long hit[kSteps];
  int mine = 0;
#pragma unroll
  for (int u = 0; u < kSteps; ++u) {
    hit[u] = __ballot(first + u * kWave < n && label != padding && id_of(raw[u], ids64, v) == label);
    mine += __popcll(hit[u]);
  }
  if (lane == 0) counts[wv] = mine;
  __syncthreads();
  int at = 0, total = 0;
  for (int w = 0; w < waves; ++w) {
    if (w < wv) at += counts[w];
    total += counts[w];
  }
#pragma unroll
  for (int u = 0; u < kSteps; ++u) {
    if (hit[u] >> lane & 1) list[at + __popcll(hit[u] & ((1ull << lane) - 1))] = static_cast<uint16_t>(first + u * kWave);
    at += __popcll(hit[u]);
  }
  __syncthreads();
  const int col = threadIdx.x & (lanes - 1), slots = blockDim.x / lanes;
  const int64_t d = groups * kV, g = blockIdx.y * static_cast<int64_t>(lanes) + col;
  float acc[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) acc[j] = 0.f;
  if (g < groups) {
    constexpr int kU = 4;   // rows in flight
    for (int i = threadIdx.x / lanes; i < total; i += kU * slots) {
      V s[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (i + u * slots < total) s[u] = reinterpret_cast<const V *>(static_cast<const T *>(grad) + list[i + u * slots] * d)[g];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (i + u * slots < total) {
#pragma unroll
          for (int j = 0; j < kV; ++j) acc[j] += static_cast<float>(s[u][j]);
        }
    }
  }
  for (int m = lanes; m < kWave; m <<= 1) {
#pragma unroll
    for (int j = 0; j < kV; ++j) acc[j] += __shfl_xor(acc[j], m, kWave);
  }
  if (lane < lanes) {
#pragma unroll
    for (int j = 0; j < kV; ++j) part[wv][lane * kV + j] = acc[j];
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < lanes && g < groups) {
    for (int w = 1; w < waves; ++w) {
#pragma unroll
      for (int j = 0; j < kV; ++j) acc[j] += part[w][lane * kV + j];
    }
    V o;
#pragma unroll
    for (int j = 0; j < kV; ++j) o[j] = static_cast<T>(acc[j] * scale);
    reinterpret_cast<V *>(static_cast<T *>(dtable) + label * d)[g] = o;
  }
}

// Columns of a tile of k_embed_few; 0: the sort and the kernels behind it.  Half tiles, for more rows at a time, where
// they fit the device at once; whole ones up to two (of fewer positions, with fewer waves, four) workgroups of 1,024
// threads per place: there it takes 0.4 to 0.8 of the others' time, at twice as many 0.5 to 1.3 of it.
int few_columns(int64_t n, int64_t v, int64_t d) {
  if (n < 1 || n > kFewMost) return 0;
  if (v * ((2 * d + kFewCols - 1) / kFewCols) <= 512) return kFewCols / 2;
  return v * ((d + kFewCols - 1) / kFewCols) <= (n <= kFewMost / 2 ? 2048 : 1024) ? kFewCols : 0;
}

template <int DT, int kV>
constexpr auto k_embed_grad_wide = &k_embed_grad<DT, kV, 4>;
template <int DT, int kV>
constexpr auto k_embed_grad_narrow = &k_embed_grad<DT, kV, 1>;
// Four rows per thread where that leaves every CU 512 threads: the pass into 32,000 rows of 512 bfloat16 columns (8,192
// positions) takes 19 us so and 22 with one, into 21 rows of 256 float32 columns (16,384 positions) 37 and 26.
bool wide_rows(int64_t v, int64_t groups) { return v * groups >= 4 * 256 * 512; }

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

dim3 row_grid(int64_t rows, dim3 block, int64_t tiles = 1) {
  const int64_t b = (rows + block.y - 1) / block.y;
  return dim3(static_cast<unsigned>(b < 65536 ? b : 65536), static_cast<unsigned>(tiles));
}

int check_embed(const char *what, int dt, int64_t n, int64_t v, int64_t d) {
  SBOD_REQUIRE(known_dt(dt), "%s: dtype %d", what, dt);
  SBOD_REQUIRE(n >= 0 && n < (1ll << 31) - 65536 && v >= 0 && v < (1ll << 31) - 65536 && d >= 0 && d < (1ll << 23),
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
  if (few_columns(n, v, d)) return align_up(1);   // (not used: a call always brings one)
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
  const int w = column_group(d, dtype, grad, grad_table);
  if (const int c = few_columns(n, v, d)) {
    const dim3 few(static_cast<unsigned>(v), static_cast<unsigned>((d + c - 1) / c));
    const dim3 threads(n <= 4 * kFewWave ? 256 : n <= 8 * kFewWave ? 512 : 1024);
    SBOD_EMBED_LAUNCH(k_embed_few, dtype, w, few, threads, grad, ids, ids64, static_cast<int>(n), v, padding, d / w, c / w, scale,
                      grad_table);
    SBOD_LAUNCHED("k_embed_few");
    return SBOD_OK;
  }
  int32_t *begin = static_cast<int32_t *>(workspace);
  int32_t *sorted = ws_at<int32_t>(workspace, align_up((v + 1) * sizeof(int32_t)));
  const int range = static_cast<int>(sort_range(v));
  const dim3 sgrid(static_cast<unsigned>((v + range - 1) / range)), sblock(kSortThreads);
  const size_t lds = static_cast<size_t>(range) * kSortWaves * sizeof(int32_t);
  if (ids64)
    hipLaunchKernelGGL(k_embed_sort<int64_t>, sgrid, sblock, lds, s, static_cast<const int64_t *>(ids), n, v, range, begin, sorted);
  else
    hipLaunchKernelGGL(k_embed_sort<int32_t>, sgrid, sblock, lds, s, static_cast<const int32_t *>(ids), n, v, range, begin, sorted);
  SBOD_LAUNCHED("k_embed_sort");
  const dim3 block = row_block(d / w);
  const int64_t tiles = (d / w + block.x - 1) / block.x;   // of a row's columns, a workgroup each
  const int rows = piece_rows(n);
  float *pieces = nullptr;
  if (n > rows) {   // (else no label can have come more often)
    const int64_t chunks = (n + rows - 1) / rows;
    pieces = ws_at<float>(workspace, align_up((v + 1) * sizeof(int32_t)) + align_up(n * sizeof(int32_t)));
    SBOD_EMBED_LAUNCH(k_embed_pieces, dtype, w, row_grid(chunks, block, tiles), block, grad, ids, ids64, begin, sorted, v, padding, chunks,
                      rows, d / w, pieces);
    SBOD_LAUNCHED("k_embed_pieces");
  }
  if (wide_rows(v, d / w))
    SBOD_EMBED_LAUNCH(k_embed_grad_wide, dtype, w, row_grid((v + 3) / 4, block, tiles), block, grad, begin, sorted, v,
                      padding, rows, d / w, pieces, scale, grad_table);
  else
    SBOD_EMBED_LAUNCH(k_embed_grad_narrow, dtype, w, row_grid(v, block, tiles), block, grad, begin, sorted, v, padding,
                      rows, d / w, pieces, scale, grad_table);
  SBOD_LAUNCHED("k_embed_grad");
  return SBOD_OK;
}
