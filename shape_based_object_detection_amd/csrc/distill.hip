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
//   w T q_v for another one, or with a bucket w T (q_o - rest) q_v / q_o.
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
  double inv_td;
};

// What a row leaves for its gradient: q_v = 2^((x - m) s - l2s); another label than the kept ones
// gets coef 2^((x - mo) s - l2so); p_k = exp((t_k - tb) / T - tl).
enum { kStM, kStL2s, kStMo, kStL2so, kStCoef, kStTb, kStTl, kStLive, kStats };

__device__ __forceinline__ bool row_has_weight(const DistillArgs &a, int64_t r) { return !a.w || a.w[r] != 0.f; }

__device__ __forceinline__ void put_row(const DistillArgs &a, int64_t r, double loss) {
  if (a.parts) a.parts[r] = loss;
  else a.rows[r] = static_cast<float>(loss);
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

// {max, sum of 2^((x - max) s)} of each chunk of a row; with a bucket, of its labels not kept.
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
    if (kBucket) mark_kept(a, r, e0, bits, kDistGran * P / 32);
    float f[kPer][P], m = kNegInf;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      ld_granule<DT>(row, e0 + static_cast<int64_t>(i * kDistThreads + threadIdx.x) * P, a.v, kNegInf, f[i]);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (kBucket) {
        const int g = i * kDistThreads + threadIdx.x;
        const uint32_t b = bits[g * P >> 5] >> (g * P & 31);
#pragma unroll
        for (int j = 0; j < P; ++j)
          if (b >> j & 1) f[i][j] = kNegInf;
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

// (the difference in 64 bits: with lse, t / T and lse are large against it)
__device__ __forceinline__ float teacher_logp(const DistillArgs &a, int64_t i, float tb, float tl) {
  return static_cast<float>((static_cast<double>(ld_any(a.top, i, a.top_dt)) - tb) * a.inv_td - tl);
}

// One wave per row: the chunks joined, the teacher's side, the row's loss and statistics.
template <int DT, bool kBucket>
__global__ __launch_bounds__(256) void k_distill_join(DistillArgs a) {
  using T = typename Elt<DT>::T;
  __shared__ int ids_s[kBucket ? 4 : 1][kBucket ? kMaxTop : 1];
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
    float m = mo, sum = so;
    int kept = 0;   // different labels kept
    if (live && kBucket) {
      for (int k = lane; k < a.k; k += kWave) {
        const int id = ld_id(a.ids, r * a.k + k, a.ids64, a.v);
        ids_s[wv][k] = id;
        if (id >= 0) m = fmaxf(m, static_cast<float>(row[id]));
      }
      m = wave_max_f32(m);
      const float base = m == kNegInf ? 0.f : m;
      wave_lds_fence();
      float sk = 0.f;
      for (int k = lane; k < a.k; k += kWave) {
        const int id = ids_s[wv][k];
        bool first = id >= 0;
        for (int j = 0; j < k && first; ++j) first = ids_s[wv][j] != id;
        if (first) {
          sk += exp2_hw((static_cast<float>(row[id]) - base) * a.s);
          ++kept;
        }
      }
      kept = wave_sum_i32(kept);
      sum = wave_sum_f32(sk) + (mo == kNegInf ? so : so * exp2_hw((mo - base) * a.s));
      wave_lds_fence();
    }
    // a row of -inf alone has no distribution: it is left out, as one of weight 0
    if (m == kNegInf && sum == 0.f) live = false;
    if (!live) {
      if (lane < kStats) st[lane] = 0.f;
      if (lane == 0) put_row(a, r, 0.0);
      continue;
    }
    const float logs = logf(sum);
    // (the few kept terms in 64 bits: a label masked by the type's lowest value is a finite loss)
    double kl = 0;
    float mass = 0.f;
    for (int k = lane; k < a.k; k += kWave) {
      const int id = ld_id(a.ids, r * a.k + k, a.ids64, a.v);
      if (id < 0) continue;
      const float logp = teacher_logp(a, r * a.k + k, tb, tl), p = expf(logp);
      const double logq = (static_cast<double>(row[id]) - m) * a.inv_td - logs;
      if (p != 0.f) kl += p * (logp - logq);   // 0 log 0 = 0
      mass += p;
    }
    kl = wave_sum_f64(kl);
    float coef = 1.f;
    if (kBucket) {
      mass = wave_sum_f32(mass);
      float rest = 1.f - mass;
      // (no label outside the kept ones: what is left of the teacher's mass is rounding)
      if (rest < 0.f || kept == a.v) rest = 0.f;
      const double logo = so == 0.f ? kNegInf : (static_cast<double>(mo) - m) * a.inv_td + logf(so) - logs;
      kl += rest > 0.f ? rest * (logf(rest) - logo) : rest;
      coef = expf(static_cast<float>(logo)) - rest;
    }
    if (lane == 0) {
      st[kStM] = m;
      st[kStL2s] = log2f(sum);
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
__global__ __launch_bounds__(256) void k_distill_weights(const float *w, int64_t n, double *parts) {
  __shared__ double red[16];
  double sum = 0;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) sum += w[i];
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
// behind a barrier, by a thread each.
template <int DT>
__global__ __launch_bounds__(kDistThreads) void k_distill_grad(DistillArgs a) {
  using T = typename Elt<DT>::T;
  constexpr int P = Elt<DT>::P, kPer = kDistGran / kDistThreads;
  __shared__ int ids_s[kMaxTop];
  __shared__ float p_s[kMaxTop];
  if (a.skip_one && *a.up == 1.f) return;   // the forward wrote this very gradient
  const int64_t items = a.n * a.nchunk;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t r = it / a.nchunk;
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
      ids_s[k] = id;
      p_s[k] = id >= 0 ? expf(teacher_logp(a, r * a.k + k, tb, tl)) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int64_t e = e0 + static_cast<int64_t>(i * kDistThreads + threadIdx.x) * P;
      ld_granule<DT>(row, e, a.v, kNegInf, f);
#pragma unroll
      for (int j = 0; j < P; ++j) f[j] = gc * exp2_hw((f[j] - mo) * a.s - l2so);
      st_granule<DT>(drow, e, a.v, aligned, f);
    }
    __syncthreads();
    for (int k = threadIdx.x; k < a.k; k += kDistThreads) {
      const int id = ids_s[k];
      if (id < 0 || id < e0 || id >= e1) continue;
      float p = 0.f;
      for (int j = 0; j < a.k; ++j) p += ids_s[j] == id ? p_s[j] : 0.f;
      const float q = exp2_hw((static_cast<float>(row[id]) - st[kStM]) * a.s - st[kStL2s]);
      drow[id] = static_cast<T>(g * (q - p));
    }
    __syncthreads();
  }
}

// A vocabulary of at most G E labels: G lanes per row hold it in registers, label j G + lane in the lane's
// slot j, so the logits are read once and the gradient written once, with the loss, in one launch.  The
// kept labels are K values beside it: lane k holds entry k (and k + G, ...), its logit gathered from the row.
// With a bucket they leave the row by a bit mask per lane; their gradients overwrite the row's.
template <int DT, int G, int E, bool kBucket>
__global__ __launch_bounds__(256) void k_distill_small(DistillArgs a) {
  using T = typename Elt<DT>::T;
  constexpr int kRows = 256 / G;
  __shared__ uint32_t masks[256];   // bit j of a lane's word: its slot j is a kept label
  __shared__ double red[16];
  if (a.skip_one && *a.up == 1.f) return;   // the forward wrote this very gradient
  const int lane = threadIdx.x % G, v = static_cast<int>(a.v), kk = a.k;
  uint32_t *mask = masks + threadIdx.x / G * G;
  mask[lane] = 0;
  const float norm = a.norm ? *a.norm : static_cast<float>(norm_of(a));
  const float up = a.up && a.up_stride == 0 ? *a.up : 1.f;
  double loss = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t r = blockIdx.x * static_cast<int64_t>(kRows) + (G == kWave ? __builtin_amdgcn_readfirstlane(threadIdx.x / G) : threadIdx.x / G);
  // a row's weight and first G entries are loaded a row ahead
  float w_next = 1.f, t_next = 0.f;
  int id_next = -1;
  const auto ahead = [&](int64_t q) {
    if (q >= a.n) return;
    if (a.w) w_next = a.w[q];
    if (lane < kk) {
      id_next = ld_id(a.ids, q * kk + lane, a.ids64, a.v);
      t_next = ld_any(a.top, q * kk + lane, a.top_dt);
    }
  };
  ahead(r);
  for (; r < a.n; r += step) {
    const T *row = static_cast<const T *>(a.x) + r * a.ldx;
    const float w = w_next, t0 = t_next;
    const int id0 = id_next;
    bool live = w != 0.f;
    // (loads first, conversions behind them: a conversion next to its load would wait for it)
    T raw[E];
    T xraw = static_cast<T>(0.f);
#pragma unroll
    for (int j = 0; j < E; ++j) raw[j] = static_cast<T>(kNegInf);
    if (live) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        if ((j + 1) * G <= v) raw[j] = row[j * G + lane];
        else if (j * G + lane < v) raw[j] = row[j * G + lane];
      }
      if (id0 >= 0) xraw = row[id0];
    }
    ahead(r + step);
    float f[E];
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] = static_cast<float>(raw[j]);
    const float x0 = static_cast<float>(xraw);
    const auto id_of = [&](int k) { return k < G ? id0 : ld_id(a.ids, r * kk + k, a.ids64, a.v); };
    const auto top_of = [&](int k) { return k < G ? t0 : ld_any(a.top, r * kk + k, a.top_dt); };
    const auto x_of = [&](int k, int id) { return k < G ? x0 : static_cast<float>(row[id]); };
    // the teacher
    float tb = 0.f, tl = 0.f;
    if (kBucket) {
      if (live) tl = a.lse[r];
    } else {
      float tm = kNegInf, sum = 0.f;
      if (live)
        for (int k = lane; k < kk; k += G)
          if (id_of(k) >= 0) tm = fmaxf(tm, top_of(k));
      tm = group_max<G>(tm);
      tb = tm == kNegInf ? 0.f : tm;
      if (live)
        for (int k = lane; k < kk; k += G)
          if (id_of(k) >= 0) sum += exp_hw((top_of(k) - tb) * a.inv_t);
      sum = group_sum<G>(sum);
      live = live && !(sum == 0.f);
      tl = log_hw(sum);
    }
    const auto logp_at = [&](float t) { return static_cast<float>((static_cast<double>(t) - tb) * a.inv_td - tl); };
    // the kept labels' bits; a label that is there already is listed twice
    bool twice = false;
    float mk = kNegInf;
    if (live)
      for (int k = lane; k < kk; k += G) {
        const int id = id_of(k);
        if (id < 0) continue;
        const uint32_t bit = 1u << (id / G);
        twice = (atomicOr(&mask[id % G], bit) & bit) || twice;
        if (kBucket) mk = fmaxf(mk, x_of(k, id));
      }
    twice = group_any<G>(twice);
    wave_lds_fence();
    const uint32_t mine = mask[lane];
    wave_lds_fence();
    mask[lane] = 0;
    // the student: the row's labels, with a bucket those not kept
    float mo = kNegInf;
    bool others = false;
    if (kBucket) {
      // (slots of the lane that hold a label: j G + lane < v)
      const int held = v > lane ? (v - lane + G - 1) / G : 0;
      others = held > 0 && (~mine & (0xffffffffu >> (32 - held))) != 0;
    }
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (kBucket && (mine >> j & 1)) f[j] = kNegInf;
      mo = fmaxf(mo, f[j]);
    }
    mo = group_max<G>(mo);
    if (kBucket) {
      mk = group_max<G>(mk);
      others = group_any<G>(others);
    }
    const float m = fmaxf(mo, mk), base = m == kNegInf ? 0.f : m, obase = mo == kNegInf ? 0.f : mo;
    float so = 0.f, sk = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      f[j] = exp2_hw((f[j] - obase) * a.s);
      so += f[j];
    }
    so = group_sum<G>(so);
    // an entry's place among those of its label: the sums' order is the list's
    const auto earlier = [&](int k, int id) {
      for (int i = 0; i < k; ++i)
        if (ld_id(a.ids, r * kk + i, a.ids64, a.v) == id) return true;
      return false;
    };
    float sum = so, mass = 0.f;
    if (kBucket) {
      if (live)
        for (int k = lane; k < kk; k += G) {
          const int id = id_of(k);
          if (id < 0) continue;
          if (!twice || !earlier(k, id)) sk += exp2_hw((x_of(k, id) - base) * a.s);
          mass += exp_hw(logp_at(top_of(k)));
        }
      sk = group_sum<G>(sk);
      mass = group_sum<G>(mass);
      sum = sk + (mo == kNegInf ? so : so * exp2_hw((mo - base) * a.s));
    }
    // a row of -inf alone has no distribution: it is left out, as one of weight 0
    live = live && !(m == kNegInf && sum == 0.f);
    const float logs = log_hw(sum);
    float coef = 1.f / sum;   // what a label not kept takes of its exponential
    double kl = 0;
    if (live) {
      // (the few kept terms in 64 bits: a label masked by the type's lowest value is a finite loss)
      for (int k = lane; k < kk; k += G) {
        const int id = id_of(k);
        if (id < 0) continue;
        const float logp = logp_at(top_of(k)), p = exp_hw(logp);
        if (p != 0.f) kl += p * (logp - ((static_cast<double>(x_of(k, id)) - base) * a.inv_td - logs));
      }
      if (kBucket) {
        float rest = 1.f - mass;
        // (no label outside the kept ones: what is left of the teacher's mass is rounding)
        if (rest < 0.f || !others) rest = 0.f;
        const double logo = so == 0.f ? kNegInf : (static_cast<double>(mo) - base) * a.inv_td + log_hw(so) - logs;
        if (lane == 0) kl += rest > 0.f ? rest * (log_hw(rest) - logo) : rest;
        coef = so == 0.f ? 0.f : (exp_hw(static_cast<float>(logo)) - rest) / so;
      }
      kl *= static_cast<double>(a.t) * a.t * w;
    }
    if (a.rows) {
      kl = group_sum<G>(kl);
      if (lane == 0) a.rows[r] = static_cast<float>(kl);
    }
    loss += kl;
    if (!a.dx) continue;
    T *drow = static_cast<T *>(a.dx) + r * a.lddx;
    float g = a.t * w * norm * up;
    if (a.up && a.up_stride) g *= a.up[r];
    const float gc = g * coef;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const T d = static_cast<T>(live ? f[j] * gc : 0.f);
      if ((j + 1) * G <= v) drow[j * G + lane] = d;
      else if (j * G + lane < v) drow[j * G + lane] = d;
    }
    wave_lds_fence();   // (the same addresses again, by the lanes that hold the entries)
    if (live)
      for (int k = lane; k < kk; k += G) {
        const int id = id_of(k);
        if (id < 0) continue;
        float p = exp_hw(logp_at(top_of(k)));
        if (twice) {
          p = 0.f;
          for (int i = 0; i < kk; ++i)
            if (ld_id(a.ids, r * kk + i, a.ids64, a.v) == id) p += exp_hw(logp_at(ld_any(a.top, r * kk + i, a.top_dt)));
        }
        drow[id] = static_cast<T>(g * (exp2_hw((x_of(k, id) - base) * a.s) / sum - p));
      }
  }
  if (a.parts) {
    loss = block_sum(loss, red);
    if (threadIdx.x == 0) a.parts[blockIdx.x] = loss;
  }
}

constexpr int kSmallMax = 2048;   // labels k_distill_small holds
constexpr int kSmallBlocks = 2048;

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
  hipLaunchKernelGGL((k_distill_join<DT, kBucket>), dim3(grid_for((a.n + 3) / 4)), dim3(256), 0, s, a);
  SBOD_LAUNCHED("k_distill_join");
  return SBOD_OK;
}

int64_t small_blocks(int64_t n, int g) {
  const int64_t b = (n + 256 / g - 1) / (256 / g);
  return b < kSmallBlocks ? b : kSmallBlocks;
}
int small_lanes(int64_t v) { return v <= 32 ? 8 : v <= 64 ? 16 : v <= 128 ? 32 : 64; }

template <int DT, bool kBucket>
int launch_small(const DistillArgs &a, hipStream_t s) {
  const int g = small_lanes(a.v);
  const dim3 grid(static_cast<unsigned>(small_blocks(a.n, g))), block(256);
#define SBOD_SMALL(G, E) hipLaunchKernelGGL((k_distill_small<DT, G, E, kBucket>), grid, block, 0, s, a)
  if (a.v <= 32) SBOD_SMALL(8, 4);
  else if (a.v <= 64) SBOD_SMALL(16, 4);
  else if (a.v <= 128) SBOD_SMALL(32, 4);
  else if (a.v <= 256) SBOD_SMALL(64, 4);
  else if (a.v <= 512) SBOD_SMALL(64, 8);
  else if (a.v <= 1024) SBOD_SMALL(64, 16);
  else if (a.v <= 1536) SBOD_SMALL(64, 24);
  else SBOD_SMALL(64, 32);
#undef SBOD_SMALL
  SBOD_LAUNCHED("k_distill_small");
  return SBOD_OK;
}

// Which kernels take a call.
enum Path { kSmall, kChunks };
Path path_of(int64_t v) { return v <= kSmallMax ? kSmall : kChunks; }

// The forward's, or with a.up the gradient's, launches of one type.
template <int DT, bool kBucket>
int launch_typed(const DistillArgs &a, hipStream_t s) {
  if (path_of(a.v) == kSmall) return launch_small<DT, kBucket>(a, s);
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
int64_t parts_count(int64_t n, int64_t v) { return path_of(v) == kSmall ? small_blocks(n, small_lanes(v)) : n; }
size_t chunks_offset(int64_t n, int64_t v) { return align_up(parts_offset() + parts_count(n, v) * sizeof(double)); }

int check_common(const char *what, const void *x, int dt, int64_t n, int64_t v, int64_t ldx, const void *ids,
                 const void *top, int top_dt, int k, float temperature, int reduction) {
  SBOD_REQUIRE(known_dt(dt) && known_dt(top_dt), "%s: dtype %d / %d", what, dt, top_dt);
  SBOD_REQUIRE(n >= 0 && v >= 1 && v < (1ll << 31) - 65536 && ldx >= v, "%s: logits [%lld, %lld] with row stride %lld",
               what, static_cast<long long>(n), static_cast<long long>(v), static_cast<long long>(ldx));
  SBOD_REQUIRE(k >= 1 && k <= kMaxTop, "%s: %d kept labels per row (1..%d)", what, k, kMaxTop);
  SBOD_REQUIRE(n < (1ll << 40) / v, "%s: %lld rows of %lld labels", what, static_cast<long long>(n), static_cast<long long>(v));
  SBOD_REQUIRE(temperature > 0.f && temperature < __builtin_inff(), "%s: temperature %g", what, temperature);
  SBOD_REQUIRE(reduction >= SBOD_REDUCE_NONE && reduction <= SBOD_REDUCE_SUM, "%s: reduction %d", what, reduction);
  SBOD_REQUIRE(n == 0 || (x && ids && top), "%s: null tensor", what);
  return SBOD_OK;
}

void set_temperature(DistillArgs &a, float t) {
  a.t = t;
  a.inv_td = 1.0 / t;
  a.inv_t = static_cast<float>(a.inv_td);
  a.s = static_cast<float>(a.inv_td * 1.44269504088896340736);
}

}  // namespace label
}  // namespace sbod

using namespace sbod;
using namespace sbod::label;

extern "C" int sbod_distill_stat_floats(void) { return kStats; }

extern "C" size_t sbod_distill_workspace_bytes(int64_t n, int64_t v, int dtype) {
  if (n < 0 || v <= 0 || !known_dt(dtype)) return 0;
  const size_t chunks = path_of(v) == kChunks ? static_cast<size_t>(n) * distill_chunks(v, dtype) * sizeof(float2) : 0;
  return chunks_offset(n, v) + chunks;
}

extern "C" int sbod_distill_fwd(const void *logits, int dtype, int64_t n, int64_t v, int64_t ld, const void *ids,
                                int ids64, const void *top, int top_dtype, int k, const float *lse,
                                const float *weights, float temperature, int reduction, float *rows, float *loss,
                                float *norm, float *stats, void *grad, int64_t grad_ld, void *workspace, size_t workspace_bytes,
                                void *stream) {
  const int bad = check_common("sbod_distill_fwd", logits, dtype, n, v, ld, ids, top, top_dtype, k, temperature, reduction);
  if (bad != SBOD_OK) return bad;
  SBOD_REQUIRE(n == 0 || ((rows || reduction != SBOD_REDUCE_NONE) && stats), "sbod_distill_fwd: null output");
  SBOD_REQUIRE(reduction == SBOD_REDUCE_NONE || (loss && norm), "sbod_distill_fwd: a reduction needs loss and norm");
  SBOD_REQUIRE(!grad || (grad_ld >= v && reduction != SBOD_REDUCE_NONE), "sbod_distill_fwd: gradient with row stride %lld, reduction %d",
               static_cast<long long>(grad_ld), reduction);
  if (workspace_bytes < sbod_distill_workspace_bytes(n, v, dtype) || !workspace) {
    set_error("sbod_distill_fwd: workspace of %zu bytes, %zu needed", workspace_bytes, sbod_distill_workspace_bytes(n, v, dtype));
    return SBOD_E_WORKSPACE;
  }
  hipStream_t s = as_stream(stream);
  DistillArgs a = {};
  a.x = logits, a.n = n, a.v = v, a.ldx = ld, a.ids = ids, a.ids64 = ids64, a.top = top, a.top_dt = top_dtype;
  a.k = k, a.lse = lse, a.w = weights, a.stats = stats, a.reduction = reduction;
  a.rows = reduction == SBOD_REDUCE_NONE ? rows : nullptr;
  a.part = ws_at<float2>(workspace, chunks_offset(n, v)), a.nchunk = distill_chunks(v, dtype);
  a.dx = grad, a.lddx = grad_ld;
  set_temperature(a, temperature);
  if (reduction != SBOD_REDUCE_NONE) a.parts = ws_at<double>(workspace, parts_offset()), a.nparts = parts_count(n, v);
  if (reduction == SBOD_REDUCE_MEAN && weights) {
    // (64 partial sums: each workgroup of the loss joins them)
    a.wparts = static_cast<const double *>(workspace);
    a.nw = static_cast<int>(n < kWeightParts * 256 ? (n + 255) / 256 : kWeightParts);
    if (n > 0) {
      hipLaunchKernelGGL(k_distill_weights, dim3(a.nw), dim3(256), 0, s, weights, n, static_cast<double *>(workspace));
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
  return grad && n > 0 && path_of(v) == kChunks ? launch_grad(a, dtype, s) : SBOD_OK;
}

extern "C" int sbod_distill_bwd(const void *logits, int dtype, int64_t n, int64_t v, int64_t ld, const void *ids,
                                int ids64, const void *top, int top_dtype, int k, const float *lse,
                                const float *weights, float temperature, int reduction, const float *norm,
                                const float *stats,
                                const float *upstream, int skip_if_one, void *grad, int64_t grad_ld, void *stream) {
  const int bad = check_common("sbod_distill_bwd", logits, dtype, n, v, ld, ids, top, top_dtype, k, temperature, reduction);
  if (bad != SBOD_OK) return bad;
  if (n == 0) return SBOD_OK;
  SBOD_REQUIRE(stats && grad && upstream && grad_ld >= v, "sbod_distill_bwd: null tensor or row stride %lld",
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
  return path_of(v) == kSmall ? launch_any(a, dtype, as_stream(stream)) : launch_grad(a, dtype, as_stream(stream));
}
