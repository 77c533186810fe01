// Distillation from a teacher's top logits (a class vocabulary's knowledge-distillation loss), with
// its gradient.
//
// For a row of student logits x [V] and the teacher's K kept (label, logit) pairs, at temperature T:
//   q = softmax(x / T);
//   without lse: p = softmax(t / T) over the kept labels, KL = sum_k p_k (log p_k - log q_k);
//   with the teacher's lse (log sum exp of its whole row / T): p_k = exp(t_k / T - lse), and the mass
//   it did not keep, rest = 1 - sum p, is one bucket against the student's mass outside the kept
//   labels, q_o: KL += rest (log rest - log q_o).
//   row loss = w T^2 KL;  d/dx_v = w T (q_v - p_v) for a kept label (p summed over its repetitions),
//   w T q_v for another one;  with a bucket w T (total q_v - p_v) and w T (total q_o - rest) q_v / q_o,
//   where total = sum p + rest: 1, unless sum p is above 1 (kept logits and lse rounded apart; rest is then
//   0) or every label is kept (there is no bucket).
//
// The other labels' sum has a maximum of its own: q_o would underflow, and 1 - sum of the kept q
// cancel, where the student is sure of a kept label.  The kept labels are gathered by themselves.
#include "label_dev.h"

namespace sbod {
namespace label {

constexpr int kMaxTop = 1024;       // kept labels per row
constexpr int kDistThreads = 256;   // k_distill_part / k_distill_grad
constexpr int kDistGran = 1024;     // 16-byte granules of a row per item: 4 per thread, 16 KB
constexpr float kNegInf = -__builtin_inff();

struct DistillArgs {
  const void *x;          // [n, v], row stride ldx
  const void *ids;        // [n, k] int32 / int64
  const void *top;        // [n, k] of top_dt
  const float *lse;       // [n] or null
  const float *w;         // [n] or null
  float *rows;            // [n] row losses (weighted); for a reduction null, and
  double *parts;          // what each row (k_distill_join) or workgroup adds to the loss, in 64 bits: a
                          // mean holds where single rows are beyond float
  const double *wparts;   // partial sums of the weights (k_distill_weights), or null
  float *stats;           // [n, kStats]
  float *loss, *norm;     // the reduced loss, and the factor on each row's gradient; null: 1
  float2 *part;           // [n, nchunk] {max, sum} of each chunk
  void *dx;               // [n, v], row stride lddx
  const float *up;        // upstream gradient, null for 1
  int64_t n, v, ldx, lddx, up_stride;
  int64_t nparts;
  int k, ids64, top_dt, nchunk, nw, reduction, skip_one;
  float t, inv_t, s;      // temperature, 1 / T, log2(e) / T
  double inv_td, tt;      // 1 / T, T^2
};

// What a row leaves for its gradient: q_v (with a bucket total q_v) = 2^((x - m) s - l2s); another label
// than the kept ones gets coef 2^((x - mo) s - l2so); p_k = exp((t_k - tb) / T - tl).
enum { kStM, kStL2s, kStMo, kStL2so, kStCoef, kStTb, kStTl, kStLive, kStats };

__device__ __forceinline__ bool row_has_weight(const DistillArgs &a, int64_t r) { return !a.w || a.w[r] != 0.f; }

__device__ __forceinline__ void put_row(const DistillArgs &a, int64_t r, double loss) {
  if (a.parts) a.parts[r] = loss;
  else a.rows[r] = static_cast<float>(loss);
}

// Where label `id` is in a table of `size` (a power of two, twice the entries at least) that holds -1 or the number
// of an entry, whose label is ids[entry]: the label's own place, or with kInsert one that now holds `k`.  An open hash:
// from the label's first place on.  (A row's entries find the repeated ones by it, each in a few steps whatever K.)
template <bool kInsert>
__device__ __forceinline__ int find_label(int *table, int size, const int *ids, int id, int k) {
  int h = static_cast<int>(static_cast<uint32_t>(id) * 2654435761u >> (__clz(size) + 1));
  for (;; h = (h + 1) & (size - 1)) {
    const int at = kInsert ? atomicCAS(&table[h], -1, k) : table[h];
    if ((kInsert && at < 0) || ids[at] == id) return h;
  }
}
__host__ __device__ inline int table_size(int k) {
  int size = 64;
  while (size < 2 * k) size *= 2;
  return size;
}

// Bits of the kept labels among the elements [e0, e0 + 32 nwords): all threads of the block.
__device__ __forceinline__ void mark_kept(const DistillArgs &a, int64_t r, int64_t e0, uint32_t *bits, int nwords) {
  for (int i = threadIdx.x; i < nwords; i += blockDim.x) bits[i] = 0;
  __syncthreads();
  for (int k = threadIdx.x; k < a.k; k += blockDim.x) {
    const int id = ld_id(a.ids, r * a.k + k, a.ids64, a.v);
    const int64_t at = id - e0;
    if (id >= 0 && at >= 0 && at < 32 * static_cast<int64_t>(nwords)) atomicOr(&bits[at >> 5], 1u << (at & 31));
  }
  __syncthreads();
}

// {max, sum of 2^((x - max) s)} of each chunk of a row; with a bucket, of its labels not kept.  For rows
// that no workgroup's registers hold: 16 KB per item, so that few long rows fill the device too.  Bound by its
// one read: 248 us for 2,048 rows of 131,072 float32 labels and a bucket (1.07 GB, 4.3 TB/s).
template <int DT, bool kBucket>
__global__ __launch_bounds__(kDistThreads) void k_distill_part(DistillArgs a) {
  using T = typename Elt<DT>::T;
  constexpr int P = Elt<DT>::P, kPer = kDistGran / kDistThreads;
  __shared__ uint32_t bits[kBucket ? kDistGran * P / 32 : 1];
  __shared__ float red[2][kDistThreads / kWave];
  const int64_t items = a.n * a.nchunk;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t r = it / a.nchunk;
    if (!row_has_weight(a, r)) continue;
    const T *row = static_cast<const T *>(a.x) + r * a.ldx;
    const int64_t e0 = (it - r * a.nchunk) * kDistGran * P - row_phase(row);
    // (whole granules are asked for together; the two that the row's ends cut, element by element)
    raw16_t raw[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int64_t e = e0 + static_cast<int64_t>(i * kDistThreads + threadIdx.x) * P;
      if (e >= 0 && e + P <= a.v) raw[i] = *reinterpret_cast<const raw16_t *>(row + e);
    }
    if (kBucket) mark_kept(a, r, e0, bits, kDistGran * P / 32);
    float f[kPer][P], m = kNegInf;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = i * kDistThreads + threadIdx.x;
      const int64_t e = e0 + static_cast<int64_t>(g) * P;
      if (e >= 0 && e + P <= a.v) raw_values<DT>(raw[i], f[i]);
      else ld_granule<DT>(row, e, a.v, kNegInf, f[i]);
      if (kBucket) {
        const uint32_t b = bits[g * P >> 5] >> (g * P & 31);
#pragma unroll
        for (int j = 0; j < P; ++j) f[i][j] = b >> j & 1 ? kNegInf : f[i][j];
      }
#pragma unroll
      for (int j = 0; j < P; ++j) m = fmaxf(m, f[i][j]);
    }
    m = wave_max_f32(m);
    const int wv = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[0][wv] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kDistThreads / kWave; ++i) m = fmaxf(m, red[0][i]);
    // (a chunk of -inf alone: its terms are 2^-inf = 0; NaN stays NaN)
    const float base = m == kNegInf ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
      for (int j = 0; j < P; ++j) sum += exp2_hw((f[i][j] - base) * a.s);
    sum = wave_sum_f32(sum);
    if ((threadIdx.x & 63) == 0) red[1][wv] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < kDistThreads / kWave; ++i) sum += red[1][i];
      a.part[it] = make_float2(m, sum);
    }
    __syncthreads();
  }
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

// One wave: the teacher's normaliser of a row, p_k = exp((t_k - tb) / T - tl); false without a kept
// label that has mass.
__device__ __forceinline__ bool teacher_norm(const DistillArgs &a, int64_t r, int lane, float *tb, float *tl) {
  if (a.lse) {
    *tb = 0.f;
    *tl = a.lse[r];
    return true;
  }
  float tm = kNegInf;
  for (int k = lane; k < a.k; k += kWave)
    if (ld_id(a.ids, r * a.k + k, a.ids64, a.v) >= 0) tm = fmaxf(tm, ld_any(a.top, r * a.k + k, a.top_dt));
  tm = wave_max_f32(tm);
  const float base = tm == kNegInf ? 0.f : tm;
  float sum = 0.f;
  for (int k = lane; k < a.k; k += kWave)
    if (ld_id(a.ids, r * a.k + k, a.ids64, a.v) >= 0)
      sum += expf((ld_any(a.top, r * a.k + k, a.top_dt) - base) * a.inv_t);
  sum = wave_sum_f32(sum);
  *tb = base;
  *tl = logf(sum);
  return !(sum == 0.f);
}

// A value that all lanes hold, in a scalar register.
__device__ __forceinline__ float uniform(float v) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}
__device__ __forceinline__ double uniform(double v) {
  return __hiloint2double(__builtin_amdgcn_readfirstlane(__double2hiint(v)), __builtin_amdgcn_readfirstlane(__double2loint(v)));
}

// The bucket of a row: the teacher's mass outside the kept labels, 1 - mass, against the student's, q_o.
// term: its part of the KL; coef: total q_o - rest.  Both sides are near 1 where the kept labels hold little, so
// their logarithms and their difference are then taken from what the kept labels hold (P - Q = q_o - rest);
// `mass` comes in 64 bits, for where they hold nearly all.  others: there is a label that is not kept (else
// what is left of the teacher's mass has no label).  total: both, 1 unless the bucket was cut off.  kOne: all lanes of a wave have one row (its values pass
// through scalar registers: k_distill_row's are full of the row).
struct Bucket {
  double term;
  float coef, total;
};
template <bool kOne>
__device__ __forceinline__ Bucket bucket_of(const DistillArgs &a, double mass, float kept, float sum, float so, float mo,
                                            float base, bool others) {
  const auto one = [](auto v) { return kOne ? uniform(v) : v; };
  mass = one(mass);
  double rest = 1.0 - mass;
  if (rest < 0 || !others) rest = 0;
  const float q = one(kept / sum);
  const bool little = q < 0.5f;
  const float logr = one(mass < 0.5 ? log1pf(static_cast<float>(-mass)) : logf(static_cast<float>(rest)));
  const double logo = so == 0.f ? kNegInf
                      : little  ? one(log1pf(-q))
                                : (static_cast<double>(mo) - base) * a.inv_td + one(logf(so)) - one(logf(sum));
  Bucket b;
  b.term = rest > 0 ? rest * (logr - logo) : rest;
  b.total = mass > 1 || !others ? static_cast<float>(mass) : 1.f;
  b.coef = little && mass < 1 && others ? static_cast<float>(mass - q)
                                        : static_cast<float>(b.total * one(expf(static_cast<float>(logo))) - rest);
  return b;
}

// (in 64 bits: with lse, t / T and lse are large against their difference)
__device__ __forceinline__ double teacher_logp(const DistillArgs &a, int64_t i, float tb, float tl) {
  return (static_cast<double>(ld_any(a.top, i, a.top_dt)) - tb) * a.inv_td - tl;
}

// One wave per row: the chunks joined, the teacher's side, the row's loss and statistics.  Bound by its chain of
// loads (ids, then the logits they name): 13 us for 2,048 rows with 64 kept labels and a bucket.
template <int DT, bool kBucket>
__global__ __launch_bounds__(256) void k_distill_join(DistillArgs a) {
  using T = typename Elt<DT>::T;
  __shared__ int ids_s[kBucket ? 4 : 1][kBucket ? kMaxTop : 1];
  extern __shared__ int tables[];   // with a bucket, table_size(K) words for each wave
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  for (int64_t r = blockIdx.x * 4ll + wv; r < a.n; r += gridDim.x * 4ll) {
    float *st = a.stats + r * kStats;
    float tb = 0.f, tl = 0.f;
    bool live = row_has_weight(a, r) && teacher_norm(a, r, lane, &tb, &tl);
    float mo = kNegInf, so = 0.f;
    if (live) {
      for (int c = lane; c < a.nchunk; c += kWave) mo = fmaxf(mo, a.part[r * a.nchunk + c].x);
      mo = wave_max_f32(mo);
      for (int c = lane; c < a.nchunk; c += kWave) {
        const float2 p = a.part[r * a.nchunk + c];
        so += p.x == kNegInf ? p.y : p.y * exp2_hw((p.x - mo) * a.s);
      }
      so = wave_sum_f32(so);
    }
    const T *row = static_cast<const T *>(a.x) + r * a.ldx;
    float m = mo, sum = so, ksum = 0.f;
    int kept = 0;   // different labels kept
    if (live && kBucket) {
      for (int k = lane; k < a.k; k += kWave) {
        const int id = ld_id(a.ids, r * a.k + k, a.ids64, a.v);
        ids_s[wv][k] = id;
        if (id >= 0) m = fmaxf(m, static_cast<float>(row[id]));
      }
      m = wave_max_f32(m);
      const float base = m == kNegInf ? 0.f : m;
      // a label listed twice counts at its first entry
      const int size = table_size(a.k);
      int *table = tables + wv * size;
      for (int i = lane; i < size; i += kWave) table[i] = -1;
      wave_lds_fence();
      for (int k = lane; k < a.k; k += kWave)
        if (ids_s[wv][k] >= 0) atomicMin(&table[find_label<true>(table, size, ids_s[wv], ids_s[wv][k], k)], k);
      wave_lds_fence();
      float sk = 0.f;
      for (int k = lane; k < a.k; k += kWave) {
        const int id = ids_s[wv][k];
        if (id >= 0 && table[find_label<false>(table, size, ids_s[wv], id, k)] == k) {
          sk += exp2_hw((static_cast<float>(row[id]) - base) * a.s);
          ++kept;
        }
      }
      kept = wave_sum_i32(kept);
      ksum = wave_sum_f32(sk);
      sum = ksum + (mo == kNegInf ? so : so * exp2_hw((mo - base) * a.s));
      wave_lds_fence();
    }
    // a row of -inf alone has no distribution, one without an entry nothing to learn: left out, as of weight 0
    if ((m == kNegInf && sum == 0.f) || (kBucket && kept == 0)) live = false;
    if (!live) {
      if (lane < kStats) st[lane] = 0.f;
      if (lane == 0) put_row(a, r, 0.0);
      continue;
    }
    const float logs = logf(sum);
    // (the few kept terms in 64 bits: a label masked by the type's lowest value is a finite loss)
    double kl = 0, mass = 0;
    float total = 1.f;
    for (int k = lane; k < a.k; k += kWave) {
      const int id = ld_id(a.ids, r * a.k + k, a.ids64, a.v);
      if (id < 0) continue;
      const double logp = teacher_logp(a, r * a.k + k, tb, tl);
      const float p = expf(static_cast<float>(logp));
      const double logq = (static_cast<double>(row[id]) - m) * a.inv_td - logs;
      if (p != 0.f) kl += p * (logp - logq);   // 0 log 0 = 0
      mass += p;
    }
    kl = wave_sum_f64(kl);
    float coef = 1.f;
    if (kBucket) {
      const Bucket b = bucket_of<true>(a, wave_sum_f64(mass), ksum, sum, so, mo, m, kept < a.v);
      kl += b.term;
      coef = b.coef, total = b.total;
    }
    if (lane == 0) {
      st[kStM] = m;
      st[kStL2s] = log2f(sum / total);
      // (no other label with mass: 2^((x - 0) s - 0) is 0 for each of them)
      st[kStMo] = so == 0.f ? 0.f : mo;
      st[kStL2so] = so == 0.f ? 0.f : log2f(so);
      st[kStCoef] = coef;
      st[kStTb] = tb;
      st[kStTl] = tl;
      st[kStLive] = 1.f;
      put_row(a, r, kl * a.t * a.t * (a.w ? a.w[r] : 1.f));
    }
  }
}

// Partial sums of the row weights, in 64 bits and a fixed order.
constexpr int kWeightParts = 64;
__global__ __launch_bounds__(1024) void k_distill_weights(const float *w, int64_t n, double *parts) {
  __shared__ double red[16];
  double sum = 0;
  const int64_t step = gridDim.x * 1024ll;
  int64_t i = blockIdx.x * 1024ll + threadIdx.x;
  for (; i + 3 * step < n; i += 4 * step) {
    const float a = w[i], b = w[i + step], c = w[i + 2 * step], d = w[i + 3 * step];
    sum += static_cast<double>(a) + b + (static_cast<double>(c) + d);
  }
  for (; i < n; i += step) sum += w[i];
  sum = block_sum(sum, red);
  if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

// The factor on each row's gradient.  All lanes of a wave.
__device__ __forceinline__ double norm_of(const DistillArgs &a) {
  if (a.reduction != SBOD_REDUCE_MEAN) return 1.0;
  if (!a.w) return 1.0 / static_cast<double>(a.n);
  const int lane = threadIdx.x & 63;
  const double w = wave_sum_f64(lane < a.nw ? a.wparts[lane] : 0.0);
  return w == 0 ? 0.0 : 1.0 / w;
}

// One block: the reduced loss of its parts, and the norm for the gradient.
__global__ __launch_bounds__(1024) void k_distill_sum(DistillArgs a) {
  __shared__ double red[16];
  double sum = 0;
  for (int64_t i = threadIdx.x; i < a.nparts; i += blockDim.x) sum += a.parts[i];
  sum = block_sum(sum, red);
  const double norm = a.n == 0 ? 0.0 : norm_of(a);
  if (threadIdx.x == 0) {
    *a.loss = static_cast<float>(norm == 0 ? 0.0 : sum * norm);
    *a.norm = static_cast<float>(norm);
  }
}

// dx of one chunk of a row from the row's statistics.  The kept labels are written a second time,
// behind a barrier, by a thread each, the masses of one listed twice added in the list's order.  The rows are
// taken from the last to the first: the ones that k_distill_part read last are still in the Infinity Cache
// (256 MB), and the gradient is stored past it.
// Bound by its read and write: 404 us for 2,048 rows of 131,072 float32 labels (2.15 GB, 5.3 TB/s); from the
// first row to the last 20 more (256 rows, all in the cache: the same both ways).
template <int DT>
__global__ __launch_bounds__(kDistThreads) void k_distill_grad(DistillArgs a) {
  using T = typename Elt<DT>::T;
  constexpr int P = Elt<DT>::P, kPer = kDistGran / kDistThreads;
  __shared__ int ids_s[kMaxTop], table[2 * kMaxTop];   // the chunk's entries (-1: another chunk's)
  __shared__ float p_s[kMaxTop];
  __shared__ int some, repeated;   // the last turn whose chunk had an entry, one listed before
  if (a.skip_one && *a.up == 1.f) return;   // the forward wrote this very gradient
  const int64_t items = a.n * a.nchunk;
  const int size = table_size(a.k);
  if (threadIdx.x == 0) some = repeated = -1;
  __syncthreads();
  int turn = 0;
  for (int64_t at = blockIdx.x; at < items; at += gridDim.x, ++turn) {
    const int64_t it = items - 1 - at, r = it / a.nchunk;
    const T *row = static_cast<const T *>(a.x) + r * a.ldx;
    T *drow = static_cast<T *>(a.dx) + r * a.lddx;
    const int phase = row_phase(row);
    const bool aligned = row_phase(drow) == phase;
    const int64_t e0 = (it - r * a.nchunk) * kDistGran * P - phase, e1 = e0 + kDistGran * P;
    const float *st = a.stats + r * kStats;
    float f[P];
    if (st[kStLive] == 0.f) {
#pragma unroll
      for (int j = 0; j < P; ++j) f[j] = 0.f;
      for (int i = 0; i < kPer; ++i)
        st_granule<DT>(drow, e0 + static_cast<int64_t>(i * kDistThreads + threadIdx.x) * P, a.v, aligned, f);
      continue;
    }
    float g = a.t * (a.w ? a.w[r] : 1.f);
    if (a.norm) g *= *a.norm;
    if (a.up) g *= a.up[r * a.up_stride];
    const float mo = st[kStMo], l2so = st[kStL2so], gc = g * st[kStCoef];
    const float tb = st[kStTb], tl = st[kStTl];
    for (int k = threadIdx.x; k < a.k; k += kDistThreads) {
      const int id = ld_id(a.ids, r * a.k + k, a.ids64, a.v);
      const bool mine = id >= 0 && id >= e0 && id < e1;
      ids_s[k] = mine ? id : -1;
      if (mine) p_s[k] = expf(static_cast<float>(teacher_logp(a, r * a.k + k, tb, tl))), some = turn;
    }
    for (int i = threadIdx.x; i < size; i += kDistThreads) table[i] = -1;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int64_t e = e0 + static_cast<int64_t>(i * kDistThreads + threadIdx.x) * P;
      ld_granule<DT>(row, e, a.v, kNegInf, f);
#pragma unroll
      for (int j = 0; j < P; ++j) f[j] = gc * exp2_hw((f[j] - mo) * a.s - l2so);
      st_granule<DT, true>(drow, e, a.v, aligned, f);
    }
    __syncthreads();
    if (some == turn) {
      for (int k = threadIdx.x; k < a.k; k += kDistThreads)
        if (ids_s[k] >= 0) atomicMin(&table[find_label<true>(table, size, ids_s, ids_s[k], k)], k);
      __syncthreads();
      const auto first_of = [&](int k) { return table[find_label<false>(table, size, ids_s, ids_s[k], k)]; };
      for (int k = threadIdx.x; k < a.k; k += kDistThreads)
        if (ids_s[k] >= 0 && first_of(k) != k) repeated = turn;
      __syncthreads();
      if (repeated == turn) {
        for (int k0 = 0; k0 < a.k; k0 += kWave) {   // a wave's entries after another's
          const int k = k0 + (threadIdx.x & 63);
          if (k0 % kDistThreads / kWave == threadIdx.x / kWave) {
            const int first = k < a.k && ids_s[k] >= 0 ? first_of(k) : k;
            for (unsigned long long late = __ballot(first != k); late; late &= late - 1) {
              if ((threadIdx.x & 63) == __ffsll(late) - 1) p_s[first] += p_s[k];
              wave_lds_fence();
            }
          }
          __syncthreads();
        }
      }
      for (int k = threadIdx.x; k < a.k; k += kDistThreads) {
        const int id = ids_s[k];
        if (id < 0 || (repeated == turn && first_of(k) != k)) continue;
        const float q = exp2_hw((static_cast<float>(row[id]) - st[kStM]) * a.s - st[kStL2s]);
        drow[id] = static_cast<T>(g * (q - p_s[k]));
      }
    }
    __syncthreads();
  }
}

// A vocabulary of at most G E labels: G lanes per row hold it in registers, label j G + lane in the lane's
// slot j, so the logits are read once and the gradient written once, with the loss, in one launch.  The
// kept labels are K values beside it: lane k holds entry k (kMore: entries from G on are taken up again where
// they are needed; their code costs the others registers), its logit gathered from the row.  A bit mask per lane says which of its slots are kept
// labels: with a bucket they leave the row's sum, and their gradients come by a table in LDS.
// Slots that every vocabulary of a (G, E) fills are read and written without a test.
// Bound by instructions and its waves' waits, not by memory: 27 us for 327,936 anchors of 21 float32 labels (8 lanes
// each; 76 MB, 2.8 TB/s; vector instructions keep the SIMDs busy 52 % of the time), 64 to 67 us for 32,768 proposals
// of 1,203 bfloat16 labels (64 lanes; 163 MB, busy 34 %).
template <int DT, int G, int E, bool kBucket, bool kMore>
__global__ __launch_bounds__(256) void k_distill_small(DistillArgs a) {
  using T = typename Elt<DT>::T;
  constexpr int kRows = 256 / G, kFull = E > 8 ? E - 8 : E == 8 ? 4 : 0;   // (launch_small)
  __shared__ uint32_t masks[256];   // bit j of a lane's word: its slot j is a kept label
  __shared__ float kept[256 * E];   // the gradients of the kept labels, at their places in the row
  __shared__ double red[16];
  if (a.skip_one && *a.up == 1.f) return;   // the forward wrote this very gradient
  const int lane = threadIdx.x % G, v = static_cast<int>(a.v), kk = a.k;
  uint32_t *mask = masks + threadIdx.x / G * G;
  float *own = kept + threadIdx.x / G * (G * E);
  mask[lane] = 0;
  const float norm = a.norm ? *a.norm : static_cast<float>(norm_of(a));
  const float up = a.up && a.up_stride == 0 ? *a.up : 1.f;
  double loss = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t r = blockIdx.x * static_cast<int64_t>(kRows) +
              (G == kWave ? __builtin_amdgcn_readfirstlane(threadIdx.x / G) : threadIdx.x / G);
  // a row's weight and first G entries are loaded a row ahead
  float w_next = 1.f;
  RawAny t_next = {};
  RawId id_next = {~0u, ~0u};
  const auto ahead = [&](int64_t q) {
    if (q >= a.n) return;
    if (a.w) w_next = a.w[q];
    const int64_t at = q * kk + min(lane, kk - 1);
    id_next = ld_raw_id(a.ids, at, a.ids64);
    t_next = ld_raw_any(a.top, at, a.top_dt);
  };
  ahead(r);
  const T *row = static_cast<const T *>(a.x) + r * a.ldx;
  T *drow = static_cast<T *>(a.dx) + r * a.lddx;
  for (; r < a.n; r += step, row += step * a.ldx, drow += step * a.lddx) {
    const float w = w_next, t0 = any_of(t_next, a.top_dt);
    const int id0 = lane < kk ? id_of(id_next, a.ids64, a.v) : -1;
    bool live = w != 0.f;
    // (all loads in one block and none used in it: they are in flight together)
    uint32_t raw[E], xraw = 0;
    if (live) {
      const auto bits = [&](int i) {   // (a 32-bit offset from the row's base)
        return *reinterpret_cast<const bits_t<DT> *>(reinterpret_cast<const char *>(row) +
                                                     static_cast<uint32_t>(i) * static_cast<uint32_t>(sizeof(T)));
      };
#pragma unroll
      for (int j = 0; j < E; ++j) raw[j] = bits(j < kFull ? j * G + lane : min(j * G + lane, v - 1));
      xraw = bits(max(id0, 0));
    }
    ahead(r + step);
    float f[E];
    if (__ballot(live) == 0) {   // no row of this wave has a weight
      if (a.rows && lane == 0) a.rows[r] = 0.f;
      if (a.dx)
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (j < kFull || j * G + lane < v) drow[j * G + lane] = static_cast<T>(0.f);
      continue;
    }
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] = live && (j < kFull || j * G + lane < v) ? bits_value<DT>(raw[j]) : kNegInf;
    const float x0 = bits_value<DT>(xraw);
    const bool has0 = live && id0 >= 0;
    // the entries from G on, of a live row: f(id, teacher's logit, student's)
    const auto more = [&](auto &&f) {
      if (kMore && live)
        for (int k = lane + G; k < kk; k += G) {
          const int id = ld_id(a.ids, r * kk + k, a.ids64, a.v);
          if (id >= 0) f(k, id, ld_any(a.top, r * kk + k, a.top_dt), static_cast<float>(row[id]));
        }
    };
    // the teacher
    float tb = 0.f, tl = 0.f;
    if (kBucket) {
      if (live) tl = a.lse[r];
    } else {
      float tm = has0 ? t0 : kNegInf, sum;
      more([&](int, int, float t, float) { tm = fmaxf(tm, t); });
      tm = group_max<G>(tm);
      tb = tm == kNegInf ? 0.f : tm;
      sum = has0 ? exp_hw((t0 - tb) * a.inv_t) : 0.f;
      more([&](int, int, float t, float) { sum += exp_hw((t - tb) * a.inv_t); });
      sum = group_sum<G>(sum);
      live = live && !(sum == 0.f);
      tl = log_hw(sum);
    }
    // (the difference in 64 bits: with lse, t / T and lse are large against it)
    const auto logp_at = [&](float t) { return static_cast<float>((static_cast<double>(t) - tb) * a.inv_td - tl); };
    // (with a bucket the masses' sum counts to the last bit: bucket_of)
    const auto p_at = [&](float logp) { return kBucket ? expf(logp) : exp_hw(logp); };
    const float logp0 = logp_at(t0), p0 = has0 ? p_at(logp0) : 0.f;
    // the kept labels' bits; a label that is there already is listed twice
    bool twice = false;
    if (has0) {
      const uint32_t bit = 1u << (id0 / G);
      twice = atomicOr(&mask[id0 % G], bit) & bit;
    }
    more([&](int, int id, float, float) {
      const uint32_t bit = 1u << (id / G);
      twice = (atomicOr(&mask[id % G], bit) & bit) || twice;
    });
    twice = group_any<G>(twice);
    wave_lds_fence();
    const uint32_t mine = mask[lane];
    wave_lds_fence();
    mask[lane] = 0;
    // A label listed twice counts at its first entry (bit c of `firsts`: this lane's entry c G + lane), and that
    // one has the sum of its masses, in the list's order, by the label's place in the row.
    uint32_t firsts = ~0u;
    if (twice) {
      uint32_t *place = reinterpret_cast<uint32_t *>(own);
      if (has0) place[id0] = ~0u;
      more([&](int, int id, float, float) { place[id] = ~0u; });
      wave_lds_fence();
      if (has0) atomicMin(&place[id0], static_cast<uint32_t>(lane));
      more([&](int k, int id, float, float) { atomicMin(&place[id], static_cast<uint32_t>(k)); });
      wave_lds_fence();
      if (has0 && place[id0] != static_cast<uint32_t>(lane)) firsts &= ~1u;
      more([&](int k, int id, float, float) {
        if (place[id] != static_cast<uint32_t>(k)) firsts &= ~(1u << (k / G));
      });
      wave_lds_fence();
      if (a.dx) {
        if (has0 && firsts & 1) own[id0] = p0;
        more([&](int k, int id, float t, float) {
          if (firsts >> (k / G) & 1) own[id] = p_at(logp_at(t));
        });
        wave_lds_fence();
        for (int c = 0; c * G < kk; ++c) {   // the others one by one
          const int k = c * G + lane;
          int id = c == 0 && has0 ? id0 : -1;
          float p = p0;
          if (kMore && c > 0 && k < kk && live) {
            id = ld_id(a.ids, r * kk + k, a.ids64, a.v);
            p = p_at(logp_at(ld_any(a.top, r * kk + k, a.top_dt)));
          }
          for (unsigned long long late = group_ballot<G>(id >= 0 && !(firsts >> c & 1)); late; late &= late - 1) {
            const int from = __ffsll(late) - 1, label = __shfl(id, from, G);
            const float more_mass = __shfl(p, from, G);
            if (lane == 0) own[label] += more_mass;
          }
        }
        wave_lds_fence();
      }
    }
    // the student: the row's labels, with a bucket those not kept
    float mo = kNegInf, mk = kNegInf;
    bool others = false;
    if (kBucket) {
      // (slots of the lane that hold a label: j G + lane < v)
      const int held = v > lane ? (v - lane + G - 1) / G : 0;
      others = group_any<G>(held > 0 && (~mine & (0xffffffffu >> (32 - held))) != 0);
      bool some = has0;
      if (has0) mk = x0;
      more([&](int, int, float, float x) { mk = fmaxf(mk, x), some = true; });
      mk = group_max<G>(mk);
      live = group_any<G>(some);   // (an entry is there in live rows only)
    }
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (kBucket && (mine >> j & 1)) f[j] = kNegInf;
      mo = fmaxf(mo, f[j]);
    }
    mo = group_max<G>(mo);
    const float m = fmaxf(mo, mk), base = m == kNegInf ? 0.f : m, obase = mo == kNegInf ? 0.f : mo;
    float so = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      f[j] = exp2_hw((f[j] - obase) * a.s);
      so += f[j];
    }
    so = group_sum<G>(so);
    const float e0 = has0 ? exp2_hw((x0 - base) * a.s) : 0.f;
    float sum = so, ksum = 0.f;
    double mass = 0;
    if (kBucket) {
      float sk = has0 && firsts & 1 ? e0 : 0.f;
      mass = p0;
      more([&](int k, int, float t, float x) {
        if (firsts >> (k / G) & 1) sk += exp2_hw((x - base) * a.s);
        mass += p_at(logp_at(t));
      });
      ksum = sk = group_sum<G>(sk);
      mass = group_sum<G>(mass);
      sum = sk + (mo == kNegInf ? so : so * exp2_hw((mo - base) * a.s));
    }
    // a row of -inf alone has no distribution: it is left out, as one of weight 0
    live = live && !(m == kNegInf && sum == 0.f);
    const float logs = log_hw(sum);
    float inv = 1.f / sum, coef = inv;   // what a label not kept takes of its exponential
    // (the few kept terms in 64 bits: a label masked by the type's lowest value is a finite loss)
    const auto term = [&](float p, float logp, float x) {   // 0 log 0 = 0
      return p == 0 ? 0.0 : p * (logp - ((static_cast<double>(x) - base) * a.inv_td - logs));
    };
    double kl = has0 ? term(p0, logp0, x0) : 0.0;
    more([&](int, int, float t, float x) { kl += term(p_at(logp_at(t)), logp_at(t), x); });
    if (kBucket) {
      const Bucket b = bucket_of<G == kWave>(a, mass, ksum, sum, so, mo, base, others);
      if (lane == 0) kl += b.term;
      inv *= b.total;
      coef = so == 0.f ? 0.f : b.coef / so;
    }
    kl = live ? kl * a.tt * w : 0.0;
    if (a.rows) {
      kl = group_sum<G>(kl);
      if (lane == 0) a.rows[r] = static_cast<float>(kl);
    }
    loss += kl;
    if (!a.dx) continue;
    float g = a.t * w * norm * up;
    if (a.up && a.up_stride) g *= a.up[r];
    if (has0 && firsts & 1) own[id0] = g * (e0 * inv - (twice ? own[id0] : p0));
    more([&](int k, int id, float t, float x) {
      if (firsts >> (k / G) & 1) own[id] = g * (exp2_hw((x - base) * a.s) * inv - (twice ? own[id] : p_at(logp_at(t))));
    });
    wave_lds_fence();
    const float gc = g * coef;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float at = own[j * G + lane], d = mine >> j & 1 ? at : f[j] * gc;
      if (j < kFull || j * G + lane < v) drow[j * G + lane] = static_cast<T>(live ? d : 0.f);
    }
    wave_lds_fence();
  }
  if (a.parts) {
    loss = block_sum(loss, red);
    if (threadIdx.x == 0) a.parts[blockIdx.x] = loss;
  }
}

constexpr int kSmallMax = 2048;   // labels k_distill_small holds
// Workgroups at most: what the device holds at once at five waves per SIMD.  (From 1,025 labels on, and with a bucket from
// 513, the registers allow two to four: a second, uneven round.)
constexpr int kSmallBlocks = 1280;

// A vocabulary that a workgroup's registers hold: NT threads with NG 16-byte granules each keep the row from
// its one read to its gradient's one write, and ask for the next row's granules as those of this one fall
// free, so that loads, exponentials and stores of a CU overlap though it holds one row at a time.  Thread k
// has kept entry k (K <= NT).  The elements before the row's first 16-byte boundary and behind its last
// granule are one value each of the first 2 P threads.
// With a bucket the kept labels leave the registers by a bit each in LDS, looked up a granule at a time.
// Bound by memory: 490 to 512 us for 4,096 rows of 131,072 bfloat16 labels (2.15 GB, 4.3 TB/s of the 5.07 that a copy
// reaches; 708 with a pass each for statistics and gradient), 552 with a bucket.  211 us for 2,049 rows of 50,001
// float32 labels and a bucket (162 us of memory), in nine rounds of 256 workgroups, the last of one row; 204 us for 4,096
// rows of 50,257 bfloat16 labels, 221 with a bucket (162 of memory).
template <int DT, bool kBucket, int NT, int NG>
__global__ __launch_bounds__(NT, NG == 16 ? 4 : 1) void k_distill_row(DistillArgs a) {
  using T = typename Elt<DT>::T;
  constexpr int P = Elt<DT>::P, NW = NT / kWave;
  constexpr uint32_t kInfBits = DT == SBOD_DT_F32 ? 0xff800000u : DT == SBOD_DT_BF16 ? 0xff80u : 0xfc00u;
  // bit e - head + P: element e is kept (head: the elements before the first granule)
  __shared__ uint32_t bits[kBucket ? NT * NG * P / 32 + 1 : 1];
  __shared__ int ids_s[NT], table[2 * NT];   // (find_label: the row's entries)
  __shared__ float top_s[NT], red[2][NW], sums[2][NW];
  // (128 registers, four waves per SIMD, have none to spare beside 16 granules: each thread's loss waits in LDS, and its
  // t is read again)
  constexpr bool kTight = NG == 16;
  __shared__ double red64[16], masses[NW], losses[kTight ? NT : 1];
  __shared__ int entered, repeated;   // the last row that has an entry (with a bucket), one listed before
                                      // (v > kSmallMax: n is below 2^31)
  if (a.skip_one && *a.up == 1.f) return;   // the forward wrote this very gradient
  const int tid = threadIdx.x, wave = tid >> 6, v = static_cast<int>(a.v), kk = a.k;
  if (kBucket)
    for (int i = tid; i < NT * NG * P / 32 + 1; i += NT) bits[i] = 0;
  table[tid] = table[tid + NT] = -1;
  if (tid == 0) entered = repeated = -1;
  __syncthreads();   // (other waves' threads write these words)
  const float norm = a.norm ? *a.norm : static_cast<float>(norm_of(a));
  const float up = a.up && a.up_stride == 0 ? *a.up : 1.f;
  double loss = 0;
  if (kTight) losses[threadIdx.x] = 0;
  const bool entry = tid < kk;
  raw16_t raw[NG];
  uint32_t xraw = 0;
  RawId idr = {};
  RawAny tr = {};
  // where a row's granules lie, and which single element this thread has (-1: none)
  const auto head_of = [&](const T *row) { return min((P - row_phase(row)) % P, v); };
  const auto single = [&](int head) {
    const int in = (v - head) / P, tail = v - head - in * P;
    return tid < head ? tid : tid >= P && tid < P + tail ? head + in * P + tid - P : -1;
  };
  // (a granule's address is a scalar base and the thread's own offset, the same for all of them)
  const uint32_t mine = static_cast<uint32_t>(tid) * 16;
  const auto base_of = [&](const T *row, int head) { return reinterpret_cast<const char *>(row + head); };
  const auto step_on = [&](const char *&at) {   // (one base that moves on, not one per granule kept)
    at += NT * 16;
    asm volatile("" : "+s"(at));
  };
  const auto fetch = [&](int i, const char *at, int left) {
    if (tid < left) raw[i] = *reinterpret_cast<const raw16_t *>(at + mine);
  };
  const auto fewer = [&](int &left) {   // (as step_on: no vector register per granule)
    left -= NT;
    asm volatile("" : "+s"(left));
  };
  // The registers hold the row as it was read, a granule's work at a time.  Without this the compiler widens
  // each element once and keeps twice the registers from pass to pass.
  const auto as_read = [&](int i) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" : "+v"(raw[i]));
  };
  const auto fetch_rest = [&](int64_t r, const T *row, int head) {
    const int e = single(head);
    if (e >= 0) xraw = reinterpret_cast<const bits_t<DT> *>(row)[e];
    if (entry) {
      idr = ld_raw_id(a.ids, r * kk + tid, a.ids64);
      tr = ld_raw_any(a.top, r * kk + tid, a.top_dt);
    }
  };
  int64_t r = blockIdx.x;
  float w_next = a.w && r < a.n ? a.w[r] : 1.f;
  if (r < a.n && w_next != 0.f) {
    const T *row = static_cast<const T *>(a.x) + r * a.ldx;
    const int head = head_of(row);
    const char *at = base_of(row, head);
#pragma unroll
    for (int i = 0, left = (v - head) / P; i < NG; ++i, step_on(at), fewer(left)) fetch(i, at, left);
    fetch_rest(r, row, head);
  }
  for (; r < a.n; r += gridDim.x) {
    const T *row = static_cast<const T *>(a.x) + r * a.ldx;
    T *drow = static_cast<T *>(a.dx) + r * a.lddx;
    const int head = head_of(row), inner = (v - head) / P, e1 = single(head);
    const bool aligned = row_phase(drow) == row_phase(row);
    const int64_t rn = r + gridDim.x;
    const T *next = static_cast<const T *>(a.x) + rn * a.ldx;
    const float w = w_next;
    w_next = a.w && rn < a.n ? a.w[rn] : 1.f;
    const bool ahead = rn < a.n && w_next != 0.f;
    const int nhead = ahead ? head_of(next) : 0, ninner = ahead ? (v - nhead) / P : 0;
    bool live = w != 0.f;
    float mo = kNegInf, so = 0.f, base = 0.f, coef = 0.f, inv = 0.f, ek = 0.f, pk = 0.f, obase = 0.f;
    int id = -1;
    if (live) {
      id = entry ? id_of(idr, a.ids64, a.v) : -1;
      const float t = any_of(tr, a.top_dt);
      uint32_t xk_raw = 0;
      if (id >= 0) xk_raw = reinterpret_cast<const bits_t<DT> *>(row)[id];
      const int place = id - head + P;
      if (entry) ids_s[tid] = id, top_s[tid] = t;
      if (kBucket && id >= 0) atomicOr(&bits[place >> 5], 1u << (place & 31)), entered = static_cast<int>(r);
      __syncthreads();
      float x1 = e1 >= 0 ? bits_value<DT>(xraw) : kNegInf;
      if (kBucket && e1 >= 0 && bits[(e1 - head + P) >> 5] >> ((e1 - head + P) & 31) & 1) x1 = kNegInf;
      // its byte in `bits`, of the first granule, and where in that (made here, not kept from row to row)
      int look = tid + 1;
      asm volatile("" : "+v"(look));
      const int shift = 4 * (look & 1);
      if (P == 4) look >>= 1;
      mo = x1;
      int left = inner;
#pragma unroll
      for (int i = 0; i < NG; ++i, fewer(left)) {
        as_read(i);
        // (by masks: a branch would hold the row twice where it joins)
        uint32_t b = 0;
        if (kBucket) {
          const uint32_t byte = reinterpret_cast<const uint8_t *>(bits)[look + i * (NT * P / 8)];
          b = P == 8 ? byte : byte >> shift & 15;
        }
        b = tid >= left ? ~0u : b;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const auto bit = [&](int k) { return static_cast<uint32_t>(static_cast<int32_t>(b << (31 - k)) >> 31); };
          const uint32_t m = DT == SBOD_DT_F32 ? bit(j) : (bit(2 * j) & 0xffffu) | bit(2 * j + 1) << 16;
          raw[i][j] = (raw[i][j] & ~m) | (m & (DT == SBOD_DT_F32 ? kInfBits : kInfBits << 16 | kInfBits));
        }
        as_read(i);
        float f[P];
        raw_values<DT>(raw[i], f);
#pragma unroll
        for (int j = 0; j < P; ++j) mo = fmaxf(mo, f[j]);
      }
      // listed before?  then the label counts at its first entry, and its masses are added in the list's order
      int h = 0;
      if (id >= 0) {
        h = find_label<true>(table, 2 * NT, ids_s, id, tid);
        atomicMin(&table[h], tid);
      }
      const float xk = bits_value<DT>(xk_raw);
      float other = id < 0 ? kNegInf : kBucket ? xk : t;   // the kept logits, or the teacher's
      mo = wave_max_f32(mo);
      other = wave_max_f32(other);
      if ((tid & 63) == 0) red[0][wave] = mo, red[1][wave] = other;
      __syncthreads();
      mo = uniform(group_max<NW>(red[0][tid % NW])), other = uniform(group_max<NW>(red[1][tid % NW]));
      if (kBucket && id >= 0) bits[place >> 5] = 0;   // (read for the last time above)
      obase = uniform(mo == kNegInf ? 0.f : mo);
      const float m = kBucket ? fmaxf(mo, other) : mo;
      base = uniform(m == kNegInf ? 0.f : m);
      const float tb = kBucket || other == kNegInf ? 0.f : other;
      float tl = kBucket ? a.lse[r] : 0.f;
      const auto logp_at = [&](float q) { return static_cast<float>((static_cast<double>(q) - tb) * a.inv_td - tl); };
      const auto p_at = [&](float logp) { return kBucket ? expf(logp) : exp_hw(logp); };
      const int entry1 = id >= 0 ? table[h] : tid;   // the label's first entry
      const bool first = id >= 0 && entry1 == tid;
      if (entry1 != tid) repeated = static_cast<int>(r);
      ids_s[tid] = entry1;   // (the labels were read for the last time before the maxima)
      ek = id >= 0 ? exp2_hw((xk - base) * a.s) : 0.f;
      float s1;         // the teacher's normaliser; with a bucket the kept labels' sum,
      double s2 = 0;    // and their mass, in 64 bits (bucket_of)
      if (kBucket) {
        s2 = pk = id >= 0 ? p_at(logp_at(t)) : 0.f;
        s1 = first ? ek : 0.f;
      } else {
        s1 = id >= 0 ? exp_hw((t - tb) * a.inv_t) : 0.f;
      }
      so = exp2_hw((x1 - obase) * a.s);
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        float f[P];
        as_read(i);
        raw_values<DT>(raw[i], f);
#pragma unroll
        for (int j = 0; j < P; ++j) so += exp2_hw((f[j] - obase) * a.s);
      }
      so = group_sum<kWave>(so), s1 = group_sum<kWave>(s1);
      if (kBucket) s2 = group_sum<kWave>(s2);
      if ((tid & 63) == 0) sums[0][wave] = so, sums[1][wave] = s1, masses[wave] = s2;
      __syncthreads();
      so = uniform(group_sum<NW>(sums[0][tid % NW])), s1 = uniform(group_sum<NW>(sums[1][tid % NW]));
      if (kBucket) s2 = group_sum<NW>(masses[tid % NW]);
      const float sum = kBucket ? s1 + (mo == kNegInf ? so : so * exp2_hw((mo - base) * a.s)) : so;
      // a row of -inf alone has no distribution, a teacher without mass, or with a bucket without an entry, nothing to
      // say: left out, as of weight 0
      live = !(m == kNegInf && sum == 0.f) && (kBucket ? entered == static_cast<int>(r) : !(s1 == 0.f));
      const float logs = log_hw(sum);
      if (!kBucket) {
        tl = log_hw(s1);
        pk = id >= 0 ? p_at(logp_at(t)) : 0.f;
      }
      inv = uniform(1.f / sum);
      coef = inv;
      // (the few kept terms in 64 bits: a label masked by the type's lowest value is a finite loss)
      double kl = pk == 0.f ? 0.0 : pk * (logp_at(kTight ? top_s[tid] : t) - ((static_cast<double>(xk) - base) * a.inv_td - logs));
      table[tid] = table[tid + NT] = -1;   // (read for the last time before the sums)
      if (repeated == static_cast<int>(r)) {
        top_s[tid] = pk;   // (this thread's own logit is read)
        __syncthreads();
        for (int w = 0; w < NW; ++w) {   // a wave's entries after another's
          if (wave == w)
            for (unsigned long long late = __ballot(ids_s[tid] != tid); late; late &= late - 1) {
              if ((tid & 63) == __ffsll(late) - 1) top_s[ids_s[tid]] += pk;
              wave_lds_fence();
            }
          __syncthreads();
        }
        pk = top_s[tid];
      }
      if (kBucket) {
        const Bucket b = bucket_of<true>(a, s2, s1, sum, so, mo, base, true);   // (K < V here)
        if (tid == 0) kl += b.term;
        inv = uniform(inv * b.total);
        coef = uniform(so == 0.f ? 0.f : b.coef / so);
      }
      kl = live ? kl * a.tt * w : 0.0;
      if (kTight) losses[tid] += kl;
      else loss += kl;
      if (a.rows) {
        kl = block_sum(kl, red64);
        if (tid == 0) a.rows[r] = static_cast<float>(kl);
      }
    } else if (a.rows && tid == 0) {
      a.rows[r] = 0.f;
    }
    float g = a.t * w * norm * up;
    if (a.up && a.up_stride) g *= a.up[r];
    const float gc = uniform(g * coef);
    if (a.dx && e1 >= 0) drow[e1] = static_cast<T>(live && !(kBucket && so == 0.f) ? gc * exp2_hw((bits_value<DT>(xraw) - obase) * a.s) : 0.f);
    const char *from = base_of(next, nhead), *to = base_of(drow, head);
    int left = inner, nleft = ninner;
#pragma unroll
    for (int i = 0; i < NG; ++i, step_on(from), step_on(to), fewer(left), fewer(nleft)) {
      if (a.dx && tid < left) {
        float f[P];
        as_read(i);
        raw_values<DT>(raw[i], f);
#pragma unroll
        for (int j = 0; j < P; ++j) f[j] = live ? gc * exp2_hw((f[j] - obase) * a.s) : 0.f;
        T *at = reinterpret_cast<T *>(const_cast<char *>(to) + mine);
        if (aligned) {
          vec_t<T, P> o;
#pragma unroll
          for (int j = 0; j < P; ++j) o[j] = static_cast<T>(f[j]);
          *reinterpret_cast<vec_t<T, P> *>(at) = o;
        } else {
#pragma unroll
          for (int j = 0; j < P; ++j) at[j] = static_cast<T>(f[j]);
        }
      }
      fetch(i, from, nleft);
    }
    __syncthreads();
    // the kept labels, over what the row's pass wrote there
    if (a.dx && live && id >= 0 && ids_s[tid] == tid) drow[id] = static_cast<T>(g * (ek * inv - pk));
    if (ahead) fetch_rest(rn, next, nhead);
  }
  if (a.parts) {
    loss = block_sum(kTight ? losses[tid] : loss, red64);
    if (tid == 0) a.parts[blockIdx.x] = loss;
  }
}

int distill_chunks(int64_t v, int dt) {
  const int64_t per = static_cast<int64_t>(kDistGran) * 16 / elt_bytes(dt);
  return static_cast<int>((v + 16 / elt_bytes(dt) - 1 + per - 1) / per);   // (a phase of P - 1 at most)
}

// A grid that walks `items`: enough workgroups for every CU many times over, far below the launch limit.
unsigned grid_for(int64_t items) { return static_cast<unsigned>(items < 65536 ? items : 65536); }

int launch_grad(const DistillArgs &a, int dt, hipStream_t s) {
  const dim3 grid(grid_for(a.n * a.nchunk)), block(kDistThreads);
  if (dt == SBOD_DT_F32)
    hipLaunchKernelGGL(k_distill_grad<SBOD_DT_F32>, grid, block, 0, s, a);
  else if (dt == SBOD_DT_BF16)
    hipLaunchKernelGGL(k_distill_grad<SBOD_DT_BF16>, grid, block, 0, s, a);
  else
    hipLaunchKernelGGL(k_distill_grad<SBOD_DT_F16>, grid, block, 0, s, a);
  SBOD_LAUNCHED("k_distill_grad");
  return SBOD_OK;
}

template <int DT, bool kBucket>
int launch_rows(const DistillArgs &a, hipStream_t s) {
  hipLaunchKernelGGL((k_distill_part<DT, kBucket>), dim3(grid_for(a.n * a.nchunk)), dim3(kDistThreads), 0, s, a);
  SBOD_LAUNCHED("k_distill_part");
  hipLaunchKernelGGL((k_distill_join<DT, kBucket>), dim3(grid_for((a.n + 3) / 4)), dim3(256),
                     kBucket ? 4 * table_size(a.k) * sizeof(int) : 0, s, a);
  SBOD_LAUNCHED("k_distill_join");
  return SBOD_OK;
}

int64_t small_blocks(int64_t n, int g) {
  const int64_t b = (n + 256 / g - 1) / (256 / g);
  return b < kSmallBlocks ? b : kSmallBlocks;
}
// Lanes per row: enough for its labels four a lane, and for its entries one a lane.
int small_lanes(int64_t v, int k) {
  int g = v <= 32 ? 8 : v <= 64 ? 16 : v <= 128 ? 32 : 64;
  while (g < 64 && g < k) g *= 2;
  return g;
}

template <int DT, bool kBucket>
int launch_small(const DistillArgs &a, hipStream_t s) {
  const int g = small_lanes(a.v, a.k);
  const dim3 grid(static_cast<unsigned>(small_blocks(a.n, g))), block(256);
#define SBOD_SMALL(G, E, MORE) hipLaunchKernelGGL((k_distill_small<DT, G, E, kBucket, MORE>), grid, block, 0, s, a)
#define SBOD_SMALL64(E) \
  do { if (a.k > 64) SBOD_SMALL(64, E, true); else SBOD_SMALL(64, E, false); } while (0)
  if (g == 8) SBOD_SMALL(8, 4, false);
  else if (g == 16) SBOD_SMALL(16, 4, false);
  else if (g == 32) SBOD_SMALL(32, 4, false);
  else if (a.v <= 256) SBOD_SMALL64(4);
  else if (a.v <= 512) SBOD_SMALL64(8);
  else if (a.v <= 1024) SBOD_SMALL64(16);
  else if (a.v <= 1536) SBOD_SMALL64(24);
  else SBOD_SMALL64(32);
#undef SBOD_SMALL64
#undef SBOD_SMALL
  SBOD_LAUNCHED("k_distill_small");
  return SBOD_OK;
}

// Threads and granules of k_distill_row for a row, smallest first, and the workgroups that the device holds at
// once.  -1: none, k_distill_part and the kernels behind it.
struct RowShape {
  int nt, ng, groups;
};
constexpr RowShape kRowShapes[] = {{256, 4, 1280}, {256, 8, 1024}, {256, 16, 1024}, {512, 16, 512}, {1024, 16, 256}};
int row_shape(int64_t v, int k, int dt) {
  const int64_t granules = v / static_cast<int64_t>(16 / elt_bytes(dt));
  for (int i = 0; i < 5; ++i)
    if (kRowShapes[i].nt >= k && static_cast<int64_t>(kRowShapes[i].nt) * kRowShapes[i].ng >= granules) return i;
  return -1;
}

// Which kernels take a call.
enum Path { kSmall, kRow, kChunks };
Path path_of(int64_t v, int k, int dt) {
  return v <= kSmallMax ? kSmall : row_shape(v, k, dt) >= 0 ? kRow : kChunks;
}
int64_t row_blocks(int64_t n, int shape) { return n < kRowShapes[shape].groups ? n : kRowShapes[shape].groups; }

template <int DT, bool kBucket>
int launch_row(const DistillArgs &a, hipStream_t s) {
  const int shape = row_shape(a.v, a.k, DT);
  const dim3 grid(static_cast<unsigned>(row_blocks(a.n, shape))), block(kRowShapes[shape].nt);
#define SBOD_ROW(I) hipLaunchKernelGGL((k_distill_row<DT, kBucket, kRowShapes[I].nt, kRowShapes[I].ng>), grid, block, 0, s, a)
  if (shape == 0) SBOD_ROW(0);
  else if (shape == 1) SBOD_ROW(1);
  else if (shape == 2) SBOD_ROW(2);
  else if (shape == 3) SBOD_ROW(3);
  else SBOD_ROW(4);
#undef SBOD_ROW
  SBOD_LAUNCHED("k_distill_row");
  return SBOD_OK;
}

// The forward's, or with a.up the gradient's, launches of one type.
template <int DT, bool kBucket>
int launch_typed(const DistillArgs &a, hipStream_t s) {
  const Path p = path_of(a.v, a.k, DT);
  if (p == kSmall) return launch_small<DT, kBucket>(a, s);
  if (p == kRow) return launch_row<DT, kBucket>(a, s);
  if (!a.up) {
    const int st = launch_rows<DT, kBucket>(a, s);
    if (st != SBOD_OK) return st;
  }
  return SBOD_OK;
}
int launch_any(const DistillArgs &a, int dt, hipStream_t s) {
  if (dt == SBOD_DT_F32) return a.lse ? launch_typed<SBOD_DT_F32, true>(a, s) : launch_typed<SBOD_DT_F32, false>(a, s);
  if (dt == SBOD_DT_BF16) return a.lse ? launch_typed<SBOD_DT_BF16, true>(a, s) : launch_typed<SBOD_DT_BF16, false>(a, s);
  return a.lse ? launch_typed<SBOD_DT_F16, true>(a, s) : launch_typed<SBOD_DT_F16, false>(a, s);
}

// The forward's workspace: partial weight sums | loss parts | chunk statistics.
size_t parts_offset() { return kWeightParts * sizeof(double); }
int64_t parts_count(int64_t n, int64_t v, int k, int dt) {
  const Path p = path_of(v, k, dt);
  return p == kSmall ? small_blocks(n, small_lanes(v, k)) : p == kRow ? row_blocks(n, row_shape(v, k, dt)) : n;
}
size_t chunks_offset(int64_t n, int64_t v, int k, int dt) {
  return align_up(parts_offset() + parts_count(n, v, k, dt) * sizeof(double));
}

int check_common(const char *what, const void *x, int dt, int64_t n, int64_t v, int64_t ldx, const void *ids,
                 const void *top, int top_dt, int k, float temperature, int reduction) {
  SBOD_REQUIRE(known_dt(dt) && known_dt(top_dt), "%s: dtype %d / %d", what, dt, top_dt);
  SBOD_REQUIRE(n >= 0 && v >= 1 && v < (1ll << 31) - 65536 && ldx >= v, "%s: logits [%lld, %lld] with row stride %lld",
               what, static_cast<long long>(n), static_cast<long long>(v), static_cast<long long>(ldx));
  SBOD_REQUIRE(k >= 1 && k <= kMaxTop, "%s: %d kept labels per row (1..%d)", what, k, kMaxTop);
  SBOD_REQUIRE(n < (1ll << 40) / v, "%s: %lld rows of %lld labels", what, static_cast<long long>(n), static_cast<long long>(v));
  SBOD_REQUIRE(temperature >= 1e-30f && temperature <= 1e30f, "%s: temperature %g", what, temperature);   // (1 / T and T^2 / T)
  SBOD_REQUIRE(reduction >= SBOD_REDUCE_NONE && reduction <= SBOD_REDUCE_SUM, "%s: reduction %d", what, reduction);
  SBOD_REQUIRE(n == 0 || (x && ids && top), "%s: null tensor", what);
  return SBOD_OK;
}

void set_temperature(DistillArgs &a, float t) {
  a.t = t;
  a.inv_td = 1.0 / t;
  a.tt = static_cast<double>(t) * t;
  a.inv_t = static_cast<float>(a.inv_td);
  a.s = static_cast<float>(a.inv_td * 1.44269504088896340736);
}

}  // namespace label
}  // namespace sbod

using namespace sbod;
using namespace sbod::label;

extern "C" int sbod_distill_stat_floats(void) { return kStats; }

extern "C" size_t sbod_distill_workspace_bytes(int64_t n, int64_t v, int k, int dtype) {
  if (n < 0 || v <= 0 || k <= 0 || k > kMaxTop || !known_dt(dtype)) return 0;
  const size_t chunks = path_of(v, k, dtype) == kChunks ? static_cast<size_t>(n) * distill_chunks(v, dtype) * sizeof(float2) : 0;
  return chunks_offset(n, v, k, dtype) + chunks;
}

extern "C" size_t sbod_distill_stats_bytes(int64_t n, int64_t v, int k, int dtype) {
  if (n < 0 || v <= 0 || k <= 0 || k > kMaxTop || !known_dt(dtype) || path_of(v, k, dtype) != kChunks) return 0;
  return static_cast<size_t>(n) * kStats * sizeof(float);
}

extern "C" int sbod_distill_fwd(const void *logits, int dtype, int64_t n, int64_t v, int64_t ld, const void *ids,
                                int ids64, const void *top, int top_dtype, int k, const float *lse,
                                const float *weights, float temperature, int reduction, float *rows, float *loss,
                                float *norm, float *stats, void *grad, int64_t grad_ld, void *workspace, size_t workspace_bytes,
                                void *stream) {
  const int bad = check_common("sbod_distill_fwd", logits, dtype, n, v, ld, ids, top, top_dtype, k, temperature, reduction);
  if (bad != SBOD_OK) return bad;
  SBOD_REQUIRE(n == 0 || ((rows || reduction != SBOD_REDUCE_NONE) && (stats || sbod_distill_stats_bytes(n, v, k, dtype) == 0)),
               "sbod_distill_fwd: null output");
  SBOD_REQUIRE(reduction == SBOD_REDUCE_NONE || (loss && norm), "sbod_distill_fwd: a reduction needs loss and norm");
  SBOD_REQUIRE(!grad || (grad_ld >= v && reduction != SBOD_REDUCE_NONE), "sbod_distill_fwd: gradient with row stride %lld, reduction %d",
               static_cast<long long>(grad_ld), reduction);
  if (workspace_bytes < sbod_distill_workspace_bytes(n, v, k, dtype) || !workspace) {
    set_error("sbod_distill_fwd: workspace of %zu bytes, %zu needed", workspace_bytes, sbod_distill_workspace_bytes(n, v, k, dtype));
    return SBOD_E_WORKSPACE;
  }
  hipStream_t s = as_stream(stream);
  DistillArgs a = {};
  a.x = logits, a.n = n, a.v = v, a.ldx = ld, a.ids = ids, a.ids64 = ids64, a.top = top, a.top_dt = top_dtype;
  a.k = k, a.lse = lse, a.w = weights, a.stats = stats, a.reduction = reduction;
  a.rows = reduction == SBOD_REDUCE_NONE ? rows : nullptr;
  a.part = ws_at<float2>(workspace, chunks_offset(n, v, k, dtype)), a.nchunk = distill_chunks(v, dtype);
  a.dx = grad, a.lddx = grad_ld;
  set_temperature(a, temperature);
  if (reduction != SBOD_REDUCE_NONE) a.parts = ws_at<double>(workspace, parts_offset()), a.nparts = parts_count(n, v, k, dtype);
  if (reduction == SBOD_REDUCE_MEAN && weights) {
    // (64 partial sums: each workgroup of the loss joins them)
    a.wparts = static_cast<const double *>(workspace);
    a.nw = static_cast<int>(n < kWeightParts * 1024 ? (n + 1023) / 1024 : kWeightParts);
    if (n > 0) {
      hipLaunchKernelGGL(k_distill_weights, dim3(a.nw), dim3(1024), 0, s, weights, n, static_cast<double *>(workspace));
      SBOD_LAUNCHED("k_distill_weights");
    }
  }
  if (n > 0) {
    const int st = launch_any(a, dtype, s);
    if (st != SBOD_OK) return st;
  }
  if (reduction == SBOD_REDUCE_NONE) return SBOD_OK;
  a.loss = loss, a.norm = norm;
  hipLaunchKernelGGL(k_distill_sum, dim3(1), dim3(1024), 0, s, a);
  SBOD_LAUNCHED("k_distill_sum");
  return grad && n > 0 && path_of(v, k, dtype) == kChunks ? launch_grad(a, dtype, s) : SBOD_OK;
}

extern "C" int sbod_distill_bwd(const void *logits, int dtype, int64_t n, int64_t v, int64_t ld, const void *ids,
                                int ids64, const void *top, int top_dtype, int k, const float *lse,
                                const float *weights, float temperature, int reduction, const float *norm,
                                const float *stats,
                                const float *upstream, int skip_if_one, void *grad, int64_t grad_ld, void *stream) {
  const int bad = check_common("sbod_distill_bwd", logits, dtype, n, v, ld, ids, top, top_dtype, k, temperature, reduction);
  if (bad != SBOD_OK) return bad;
  if (n == 0) return SBOD_OK;
  SBOD_REQUIRE((stats || sbod_distill_stats_bytes(n, v, k, dtype) == 0) && grad && upstream && grad_ld >= v,
               "sbod_distill_bwd: null tensor or row stride %lld",
               static_cast<long long>(grad_ld));
  SBOD_REQUIRE(reduction == SBOD_REDUCE_NONE || norm, "sbod_distill_bwd: a reduction needs the forward's norm");
  SBOD_REQUIRE(!skip_if_one || reduction != SBOD_REDUCE_NONE, "sbod_distill_bwd: skip_if_one needs a reduction");
  DistillArgs a = {};
  a.x = logits, a.n = n, a.v = v, a.ldx = ld, a.ids = ids, a.ids64 = ids64, a.top = top, a.top_dt = top_dtype;
  a.k = k, a.lse = lse, a.w = weights, a.reduction = reduction, a.skip_one = skip_if_one;
  a.norm = reduction == SBOD_REDUCE_NONE ? nullptr : const_cast<float *>(norm);
  a.stats = const_cast<float *>(stats), a.up = upstream, a.up_stride = reduction == SBOD_REDUCE_NONE ? 1 : 0;
  a.nchunk = distill_chunks(v, dtype), a.dx = grad, a.lddx = grad_ld;
  set_temperature(a, temperature);
  return path_of(v, k, dtype) != kChunks ? launch_any(a, dtype, as_stream(stream)) : launch_grad(a, dtype, as_stream(stream));
}
