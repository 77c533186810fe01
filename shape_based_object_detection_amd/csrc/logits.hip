// Penalties for repeated labels, biases and masks on the logits that a decoder is about to choose from.
//
// For a row x [V] with a history of labels, its first `prompt` entries given and the rest answered:
//   x_v -> x_v / r (x_v > 0) or x_v r, where v is in the history;
//   x_v -> x_v - frequency count_v - presence [count_v > 0], count over the answered entries;
//   x_v -> x_v + bias_v (+ every listed bias of v, in the order listed);
//   x_v -> -inf where the mask forbids v.
// In 32 bits, one rounding at the end.
#include "label_dev.h"

namespace sbod {
namespace label {

constexpr int kLogThreads = 256;
constexpr int kLogTile = 4096;            // labels per item: their counts and listed biases in LDS, 32 KB
constexpr uint32_t kSeen = 0x80000000u;   // in the history's given part; the low bits count the answers

struct LogitsArgs {
  const void *x;
  void *out;
  const void *hist;             // [n, len] int32 / int64, row stride ldh
  const int32_t *hist_len, *prompt_len;   // [n] or null
  const float *rep, *pres, *freq;         // [n] or null: the scalars below
  const void *bias;             // [n, v] of bias_dt, row stride ldb (0: one row)
  const void *bias_ids;         // [n, m] int32 / int64, row stride ldi (0: one row)
  const float *bias_val;        // [n, m], row stride ldv
  const void *mask;             // bits: int32 words; bytes: truth values; row stride ldm in elements
  int64_t n, v, ldx, ldo, ldh, ldb, ldi, ldv, ldm;
  int64_t len;
  int m, hist64, ids64, bias_dt, mask_kind, ntile;
  float rep_s, pres_s, freq_s;
};

template <int DT>
__global__ __launch_bounds__(kLogThreads) void k_logits(LogitsArgs a) {
  using T = typename Elt<DT>::T;
  constexpr int P = Elt<DT>::P;
  __shared__ uint32_t cnt[kLogTile];
  __shared__ float add[kLogTile];
  const int64_t items = a.n * a.ntile;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t r = it / a.ntile;
    const T *row = static_cast<const T *>(a.x) + r * a.ldx;
    T *orow = static_cast<T *>(a.out) + r * a.ldo;
    const int phase = row_phase(row);
    const bool aligned = row_phase(orow) == phase;
    const int64_t e0 = (it - r * a.ntile) * kLogTile - phase;
    int64_t len = a.len;
    if (a.hist_len) len = min(len, static_cast<int64_t>(max(a.hist_len[r], 0)));
    const int64_t given = a.prompt_len ? a.prompt_len[r] : 0;
    for (int i = threadIdx.x; i < kLogTile; i += kLogThreads) {
      cnt[i] = 0;
      add[i] = 0.f;
    }
    __syncthreads();
    for (int64_t i = threadIdx.x; i < len; i += kLogThreads) {
      const int id = ld_id(a.hist, r * a.ldh + i, a.hist64, a.v);
      const int64_t at = id - e0;
      if (id < 0 || at < 0 || at >= kLogTile) continue;
      if (i < given)
        atomicOr(&cnt[at], kSeen);
      else
        atomicAdd(&cnt[at], 1u);
    }
    for (int i = threadIdx.x; i < a.m; i += kLogThreads) {
      const int id = ld_id(a.bias_ids, r * a.ldi + i, a.ids64, a.v);
      const int64_t at = id - e0;
      if (id < 0 || at < 0 || at >= kLogTile) continue;
      // the first of a repeated label's entries adds them all, in order
      bool first = true;
      for (int j = 0; j < i && first; ++j) first = ld_id(a.bias_ids, r * a.ldi + j, a.ids64, a.v) != id;
      if (!first) continue;
      float s = 0.f;
      for (int j = i; j < a.m; ++j)
        if (ld_id(a.bias_ids, r * a.ldi + j, a.ids64, a.v) == id) s += a.bias_val[r * a.ldv + j];
      add[at] = s;
    }
    __syncthreads();
    const float rep = a.rep ? a.rep[r] : a.rep_s, pres = a.pres ? a.pres[r] : a.pres_s,
                freq = a.freq ? a.freq[r] : a.freq_s;
    for (int g = threadIdx.x; g < kLogTile / P; g += kLogThreads) {
      const int64_t e = e0 + static_cast<int64_t>(g) * P;
      if (e >= a.v) break;
      float f[P];
      ld_granule<DT>(row, e, a.v, 0.f, f);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        if (e + j < 0 || e + j >= a.v) continue;
        const uint32_t c = cnt[g * P + j];
        if (c) {
          f[j] = f[j] > 0.f ? f[j] / rep : f[j] * rep;
          const uint32_t answered = c & ~kSeen;
          f[j] = f[j] - freq * static_cast<float>(answered);
          if (answered) f[j] -= pres;
        }
        if (a.bias) f[j] += ld_any(a.bias, r * a.ldb + e + j, a.bias_dt);
        f[j] += add[g * P + j];
        bool ok = true;
        if (a.mask_kind == SBOD_MASK_BITS)
          ok = static_cast<const uint32_t *>(a.mask)[r * a.ldm + ((e + j) >> 5)] >> ((e + j) & 31) & 1;
        else if (a.mask_kind == SBOD_MASK_BYTES)
          ok = static_cast<const uint8_t *>(a.mask)[r * a.ldm + e + j] != 0;
        if (!ok) f[j] = -__builtin_inff();
      }
      st_granule<DT>(orow, e, a.v, aligned, f);
    }
    __syncthreads();
  }
}

}  // namespace label
}  // namespace sbod

using namespace sbod;
using namespace sbod::label;

extern "C" int sbod_logits_process(const void *logits, int dtype, int64_t n, int64_t v, int64_t ld, const void *history,
                                   int history64, int64_t history_cols, int64_t history_ld, const int32_t *history_len,
                                   const int32_t *prompt_len, const float *repetition, const float *presence,
                                   const float *frequency, float repetition_all, float presence_all,
                                   float frequency_all, const void *bias, int bias_dtype, int64_t bias_ld,
                                   const void *bias_ids, int bias_ids64, const float *bias_values, int bias_cols,
                                   int64_t bias_ids_ld, int64_t bias_values_ld, const void *mask, int mask_kind,
                                   int64_t mask_ld, void *out, int64_t out_ld, void *stream) {
  SBOD_REQUIRE(known_dt(dtype) && (!bias || known_dt(bias_dtype)), "sbod_logits_process: dtype %d / %d", dtype, bias_dtype);
  SBOD_REQUIRE(n >= 0 && v >= 1 && v < (1ll << 31) - 65536 && ld >= v && out_ld >= v && n < (1ll << 40) / v,
               "sbod_logits_process: logits [%lld, %lld], row strides %lld / %lld", static_cast<long long>(n),
               static_cast<long long>(v), static_cast<long long>(ld), static_cast<long long>(out_ld));
  SBOD_REQUIRE(history_cols >= 0 && history_cols < (1ll << 31) && bias_cols >= 0 && history_ld >= 0 && bias_ld >= 0 &&
                   bias_ids_ld >= 0 && bias_values_ld >= 0 && mask_ld >= 0,
               "sbod_logits_process: negative size or stride");
  SBOD_REQUIRE(mask_kind == SBOD_MASK_NONE || ((mask_kind == SBOD_MASK_BITS || mask_kind == SBOD_MASK_BYTES) && mask),
               "sbod_logits_process: mask kind %d", mask_kind);
  SBOD_REQUIRE((history_cols == 0 || history) && (bias_cols == 0 || (bias_ids && bias_values)),
               "sbod_logits_process: null history or listed bias");
  SBOD_REQUIRE(repetition || repetition_all > 0.f, "sbod_logits_process: repetition %g", repetition_all);
  if (n == 0) return SBOD_OK;
  SBOD_REQUIRE(logits && out, "sbod_logits_process: null tensor");
  LogitsArgs a = {};
  a.x = logits, a.out = out, a.n = n, a.v = v, a.ldx = ld, a.ldo = out_ld;
  a.hist = history, a.hist64 = history64, a.len = history_cols, a.ldh = history_ld, a.hist_len = history_len;
  a.prompt_len = prompt_len, a.rep = repetition, a.pres = presence, a.freq = frequency;
  a.rep_s = repetition_all, a.pres_s = presence_all, a.freq_s = frequency_all;
  a.bias = bias, a.bias_dt = bias_dtype, a.ldb = bias_ld, a.bias_ids = bias_ids, a.ids64 = bias_ids64;
  a.bias_val = bias_values, a.m = bias_cols, a.ldi = bias_ids_ld, a.ldv = bias_values_ld;
  a.mask = mask, a.mask_kind = mask_kind, a.ldm = mask_ld;
  a.ntile = static_cast<int>((v + 16 / elt_bytes(dtype) - 1 + kLogTile - 1) / kLogTile);
  const int64_t items = n * a.ntile;
  const dim3 grid(static_cast<unsigned>(items < 65536 ? items : 65536)), block(kLogThreads);
  hipStream_t s = as_stream(stream);
  if (dtype == SBOD_DT_F32)
    hipLaunchKernelGGL(k_logits<SBOD_DT_F32>, grid, block, 0, s, a);
  else if (dtype == SBOD_DT_BF16)
    hipLaunchKernelGGL(k_logits<SBOD_DT_BF16>, grid, block, 0, s, a);
  else
    hipLaunchKernelGGL(k_logits<SBOD_DT_F16>, grid, block, 0, s, a);
  SBOD_LAUNCHED("k_logits");
  return SBOD_OK;
}
