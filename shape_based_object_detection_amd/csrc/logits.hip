// Penalties for repeated labels, biases and masks on the logits that a decoder is about to choose from.
//
// For a row x [V] with a history of labels, its first `prompt` entries given and the rest answered:
//   x_v -> x_v / r (x_v > 0) or x_v r, where v is in the history;
//   x_v -> x_v - frequency count_v - presence, where v was answered, count_v times;
//   x_v -> x_v + bias_v (+ every listed bias of v, in the order listed);
//   x_v -> -inf where the mask forbids v.
// In 32 bits, one rounding at the end.
#include "label_dev.h"

namespace sbod {
namespace label {

constexpr int kLogTile = 8192;      // labels per item
constexpr int kLogThreads = 512;
constexpr int kMaxBiases = 4096;    // listed per row: 32 of the fewest threads' (sbod_logits_process)
// A label's word in the table: seen in the history's given part, with a listed bias, with two; and below
// them how often it was answered.
constexpr uint32_t kSeen = 1u << 31, kBiased = 1u << 30, kTwice = 1u << 29, kCount = kTwice - 1;

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
  int m, hist64, ids64, bias_dt, mask_kind, ntile, tile;   // tile: labels of an item, a multiple of 32
  float rep_s, pres_s, freq_s;
};

// A touched label's value but for its mask: x with the history's word of it, its bias and its listed biases' sum.
template <int kBias>
__device__ __forceinline__ float adjust(const LogitsArgs &a, int64_t r, int v, float x, uint32_t word, float listed,
                                        float rep, float pres, float freq) {
  if (word & (kSeen | kCount)) {
    x = x > 0.f ? x / rep : x * rep;
    const uint32_t answered = word & kCount;
    if (answered) x = x - freq * static_cast<float>(answered) - pres;   // (an infinite penalty times 0 is NaN)
  }
  if (kBias >= 0) x += ld_any(a.bias, r * a.ldb + v, kBias);
  return word & kBiased ? x + listed : x;
}

// P biases of type BT of the labels [e, e + P), all inside the row: in flight until bias_values.
template <int BT, int P>
struct RawBias {
  static constexpr int kWords = P * (BT == SBOD_DT_F32 ? 4 : 2) / 4;
  uint32_t w[kWords];
};
template <int BT, int P>
__device__ __forceinline__ void ld_raw_bias(RawBias<BT, P> &b, const LogitsArgs &a, int64_t r, int64_t e) {
  typedef uint32_t words_t __attribute__((ext_vector_type(RawBias<BT, P>::kWords), aligned(sizeof(typename Elt<BT>::T))));
  const words_t v = *reinterpret_cast<const words_t *>(static_cast<const typename Elt<BT>::T *>(a.bias) + r * a.ldb + e);
#pragma unroll
  for (int i = 0; i < RawBias<BT, P>::kWords; ++i) b.w[i] = v[i];   // (a load at any address)
}
template <int BT, int P>
__device__ __forceinline__ void bias_values(const RawBias<BT, P> &b, float (&f)[P]) {
#pragma unroll
  for (int j = 0; j < P; ++j)
    f[j] = BT == SBOD_DT_F32 ? __uint_as_float(b.w[j]) : bits_value<BT>(b.w[j / 2] >> (16 * (j & 1)) & 0xffff);
}

template <int kMask>
__device__ __forceinline__ bool forbidden(const LogitsArgs &a, int64_t r, int64_t v) {
  if (kMask == SBOD_MASK_BITS) return !(static_cast<const uint32_t *>(a.mask)[r * a.ldm + (v >> 5)] >> (v & 31) & 1);
  if (kMask == SBOD_MASK_BYTES) return static_cast<const uint8_t *>(a.mask)[r * a.ldm + v] == 0;
  return false;
}

// P mask bits of the labels [e, e + P), all inside the row.
template <int kMask, int P>
__device__ __forceinline__ uint32_t mask_of(const LogitsArgs &a, int64_t r, int64_t e) {
  if (kMask == SBOD_MASK_BITS) {
    const uint32_t *w = static_cast<const uint32_t *>(a.mask) + r * a.ldm;
    const uint64_t two = static_cast<uint64_t>(w[(e + P - 1) >> 5]) << 32 | w[e >> 5];
    return static_cast<uint32_t>(two >> (e & 31));   // (one word twice where they are the same: its upper copy is not reached)
  }
  if (kMask == SBOD_MASK_BYTES) {
    const uint8_t *b = static_cast<const uint8_t *>(a.mask) + r * a.ldm + e;
    uint32_t bits = 0;
    uint32_t word[P / 4];
    __builtin_memcpy(word, b, P);   // (a load at any address)
#pragma unroll
    for (int j = 0; j < P; ++j) bits |= (word[j / 4] >> (8 * (j % 4)) & 0xff) != 0 ? 1u << j : 0;
    return bits;
  }
  return ~0u;
}

// A value made where it is used: what is computed from it is not kept in registers from item to item.
__device__ __forceinline__ int here(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Elements of the list of listed labels: with room for a float for every two of m.
__host__ __device__ inline int list_size(int tile, int m) { return m > tile ? (m + 31) / 32 * 32 : tile; }

// The listed biases of a tile's labels that are listed twice (bits in `repeated`), each label's added to its place in
// `sums` (floats) in the order listed.  All threads: a wave has the places of its number modulo the waves, and reads the
// whole list, 64 entries at a time: one row of 32,000 labels and 4,096 listed biases takes 12 us, 26 where one label is
// listed twice, 100 where they are all of one.
__device__ __forceinline__ void sum_repeated(const LogitsArgs &a, int64_t r, int64_t e0, uint32_t *sums, const uint32_t *repeated) {
  const int me = here(threadIdx.x), lane = me & 63, wave = __builtin_amdgcn_readfirstlane(me >> 6), waves = blockDim.x >> 6;
  const auto one = [](int v, int l) { return __builtin_amdgcn_readlane(v, l); };
  const auto id_at = [&](int i) { return ld_raw_id(a.bias_ids, r * a.ldi + min(i, a.m - 1), a.ids64); };
  const auto value_at = [&](int i) { return a.bias_val[r * a.ldv + min(i, a.m - 1)]; };
  RawId next = id_at(lane);
  float next_value = value_at(lane);
  for (int i = lane; i - lane < a.m; i += kWave) {
    const int id = i < a.m ? id_of(next, a.ids64, a.v) : -1;
    const float value = next_value;
    next = id_at(i + kWave), next_value = value_at(i + kWave);
    const int64_t off = id - e0;
    const int at = id >= 0 && off >= 0 && off < a.tile ? static_cast<int>(off) : 0;
    const bool mine = id >= 0 && off == at && (at & (waves - 1)) == wave && (repeated[at >> 5] >> (at & 31) & 1);
    unsigned long long todo = __ballot(mine), same = todo;   // same: the lanes that have this one's label
    if (todo == 0) continue;
    for (int b = 0; 1 << b < a.tile; ++b) {
      const unsigned long long set = __ballot(at >> b & 1);
      same &= at >> b & 1 ? set : ~set;
    }
    const bool alone = mine && (same & (same - 1)) == 0;
    if (alone) sums[at] = __float_as_uint(__uint_as_float(sums[at]) + value);
    for (todo &= ~__ballot(alone); todo;) {   // a label's lanes one after another
      const int from = __ffsll(todo) - 1, to = one(at, from);
      unsigned long long group = static_cast<uint32_t>(one(static_cast<int>(same >> 32), from));
      group = group << 32 | static_cast<uint32_t>(one(static_cast<int>(same), from));
      todo &= ~group;
      float sum = __uint_as_float(sums[to]);
      if (group == ~0ull) {   // (lists filled up with one label: each lane's number is in the instruction)
#pragma unroll
        for (int l = 0; l < kWave; ++l) sum += __int_as_float(one(__float_as_int(value), l));
      } else {
        for (; group; group &= group - 1) sum += __int_as_float(one(__float_as_int(value), __ffsll(group) - 1));
      }
      if (lane == from) sums[to] = __float_as_uint(sum);
    }
    wave_lds_fence();
  }
}

// An item is a row's tile of up to kLogTile labels.  Its logits are on their way while the history is read:
// the answers' counts go to a table of the tile in LDS (integer atomics), the first touch of a label puts it
// on a list, and the first of its listed biases' threads owns it.  Each touched label is then computed by one
// thread, its value taking its word's place in the table, and the tile passes through registers once, the
// touched labels (a bit each) from the table.  Labels with two listed biases or more are written again behind
// that, when the registers are free (sum_repeated).  What bounds it is the chain of those steps at the workgroups
// that a CU's LDS holds (three): loads are asked for before the step that they wait behind.  53 us for 256 rows of
// 131,072 bfloat16 labels with up to 4,096 entries, 300 listed biases and a bit mask (142 MB: 2.7 TB/s); without
// history and biases 29.  One row of 32,000 float32 labels: 6 us.  Every tile reads its row's whole history, one row of
// 131,072 labels takes 7 us with 4,096 entries, 77 with 131,072 and 445 with 1,048,576.
template <int DT, int kMask, int kBias>
__global__ __launch_bounds__(kLogThreads) void k_logits(LogitsArgs a) {
  using T = typename Elt<DT>::T;
  constexpr int BT = kBias < 0 ? SBOD_DT_F32 : kBias;
  constexpr int P = Elt<DT>::P, kPer = kLogTile / P / kLogThreads;
  // [a.tile] words, then values; [a.tile] listed labels; twice [a.tile] bits; [a.m / 2] words and labels of the labels
  // with two listed biases.  Their logits take the list's place (list_size)
  extern __shared__ __attribute__((aligned(16))) uint32_t table[];
  __shared__ int listed, repeats;
  uint16_t *list = reinterpret_cast<uint16_t *>(table + a.tile);
  uint8_t *touched = reinterpret_cast<uint8_t *>(list + list_size(a.tile, a.m));
  uint32_t *owned = reinterpret_cast<uint32_t *>(touched + a.tile / 8);   // labels with a listed bias
  uint32_t *words = owned + a.tile / 32;
  uint16_t *places = reinterpret_cast<uint16_t *>(words + a.m / 2);
  const int nt = blockDim.x;
  const int64_t items = a.n * a.ntile;
  const bool build = a.len > 0 || a.m > 0;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int lane = here(threadIdx.x);
    // (a row's tiles one after another, on different XCDs: on one XCD they wait for the same lines of the row's
    // history, 76 against 61 us for 256 rows of 131,072 labels with up to 4,096 entries)
    const int64_t r = it / a.ntile, t = it - r * a.ntile;
    const T *row = static_cast<const T *>(a.x) + r * a.ldx;
    T *orow = static_cast<T *>(a.out) + r * a.ldo;
    const int phase = row_phase(row);
    const bool aligned = row_phase(orow) == phase;
    const int64_t e0 = t * kLogTile - phase;
    if (e0 >= a.v) continue;   // (a last tile that only other rows' starts reach into)
    raw16_t raw[kPer];
    uint32_t ok[kPer];
    RawBias<BT, P> rb[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int64_t e = e0 + static_cast<int64_t>(i * nt + lane) * P;
      if (i * nt + lane < a.tile / P && e >= 0 && e + P <= a.v) {
        raw[i] = *reinterpret_cast<const raw16_t *>(row + e);
        ok[i] = mask_of<kMask, P>(a, r, e);
        if (kBias >= 0) ld_raw_bias<BT, P>(rb[i], a, r, e);
      }
    }
    if (build) {
      // what the row brings is asked for at once: the first entries before the history's length is known
      constexpr int kU = 2;
      RawId id[kU], bid = {};
      float bval = 0.f, bx = 0.f;
      int64_t len = a.len;
      const auto hist = [&](int64_t i) { return ld_raw_id(a.hist, r * a.ldh + min(i, a.len - 1), a.hist64); };
      if (a.m > 0) {
        bid = ld_raw_id(a.bias_ids, r * a.ldi + min(lane, a.m - 1), a.ids64);
        bval = a.bias_val[r * a.ldv + min(lane, a.m - 1)];
      }
      if (a.len > 0) {
#pragma unroll
        for (int u = 0; u < kU; ++u) id[u] = hist(u * nt + lane);
      }
      const int32_t lim = a.hist_len ? a.hist_len[r] : 0, prompt = a.prompt_len ? a.prompt_len[r] : 0;
      const float rep = a.rep ? a.rep[r] : a.rep_s, pres = a.pres ? a.pres[r] : a.pres_s,
                  freq = a.freq ? a.freq[r] : a.freq_s;
      for (int i = lane; i < a.tile / 4; i += nt) reinterpret_cast<raw16_t *>(table)[i] = raw16_t{0, 0, 0, 0};
      for (int i = lane; i < a.tile / 16; i += nt) reinterpret_cast<uint32_t *>(touched)[i] = 0;   // (owned with it)
      if (lane == 0) listed = repeats = 0;
      if (a.hist_len) len = min(len, static_cast<int64_t>(max(lim, 0)));
      const auto place = [&](int label) {   // in the tile, or -1
        const int64_t at = label - e0;
        return label >= 0 && at >= 0 && at < a.tile ? static_cast<int>(at) : -1;
      };
      const int bat = lane < a.m ? place(id_of(bid, a.ids64, a.v)) : -1;
      if (bat >= 0) bx = static_cast<float>(row[e0 + bat]);
      __syncthreads();
      const auto mark = [&](int at) { atomicOr(reinterpret_cast<uint32_t *>(touched) + (at >> 5), 1u << (at & 31)); };
      for (int64_t i = lane; i - lane < len; i += kU * nt) {
        RawId next[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) next[u] = hist(i + (kU + u) * nt);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int at = i + u * nt < len ? place(id_of(id[u], a.hist64, a.v)) : -1;
          id[u] = next[u];
          if (at < 0) continue;
          const uint32_t was = i + u * nt < prompt ? atomicOr(&table[at], kSeen) : atomicAdd(&table[at], 1u);
          if (was == 0) {
            list[atomicAdd(&listed, 1)] = static_cast<uint16_t>(at);
            mark(at);
          }
        }
      }
      uint32_t own = 0;   // which of this thread's listed biases own their labels (at most 32: launch)
      const auto biased = [&](int i) {
        return i == lane ? bat : place(ld_id(a.bias_ids, r * a.ldi + i, a.ids64, a.v));
      };
      for (int i = lane, c = 0; i < a.m; i += nt, ++c) {
        const int at = biased(i);
        if (at < 0) continue;
        if (atomicOr(&table[at], kBiased) & kBiased) {
          if (!(atomicOr(&table[at], kTwice) & kTwice)) places[atomicAdd(&repeats, 1)] = static_cast<uint16_t>(at);
        } else {
          own |= 1u << c;
          mark(at);
          atomicOr(&owned[at >> 5], 1u << (at & 31));
        }
      }
      __syncthreads();
      const auto settle = [&](int at, float x, float bias) {
        const uint32_t word = table[at];
        if (word & kTwice) return;   // (below)
        x = adjust<kBias>(a, r, static_cast<int>(e0 + at), x, word, bias, rep, pres, freq);
        table[at] = __float_as_uint(x);
      };
      for (int i = lane; i < listed; i += nt) {
        const int at = list[i];
        if (!(owned[at >> 5] >> (at & 31) & 1)) settle(at, static_cast<float>(row[e0 + at]), 0.f);
      }
      if (own & 1) settle(bat, bx, bval);
      for (int i = lane + nt, c = 1; i < a.m; i += nt, ++c)
        if (own >> c & 1) settle(biased(i), static_cast<float>(row[e0 + biased(i)]), a.bias_val[r * a.ldv + i]);
      __syncthreads();
      if (repeats > 0) {   // (a.m / 2 at most; `out` may be the logits)
        for (int i = lane; i < repeats; i += nt) reinterpret_cast<float *>(list)[i] = static_cast<float>(row[e0 + places[i]]);
        __syncthreads();
      }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = i * nt + lane;
      const int64_t e = e0 + static_cast<int64_t>(g) * P;
      if (g >= a.tile / P || e >= a.v) break;
      const uint32_t bits = !build ? 0 : P == 8 ? touched[g] : touched[g / 2] >> (4 * (g & 1)) & 15;
      if (e >= 0 && e + P <= a.v) {
        float f[P];
        raw_values<DT>(raw[i], f);
        if (kBias >= 0) {
          float bias[P];
          bias_values<BT, P>(rb[i], bias);
#pragma unroll
          for (int j = 0; j < P; ++j) f[j] += bias[j];
        }
        if (bits) {
#pragma unroll
          for (int j = 0; j < P; j += 4) {
            const raw16_t w = reinterpret_cast<const raw16_t *>(table)[(g * P + j) / 4];
#pragma unroll
            for (int c = 0; c < 4; ++c) f[j + c] = bits >> (j + c) & 1 ? __uint_as_float(w[c]) : f[j + c];
          }
        }
#pragma unroll
        for (int j = 0; j < P; ++j)
          if (kMask != SBOD_MASK_NONE && !(ok[i] >> j & 1)) f[j] = -__builtin_inff();
        st_granule<DT>(orow, e, a.v, aligned, f);
      } else {   // a granule that the row's start or end cuts
        for (int j = 0; j < P; ++j) {
          if (e + j < 0 || e + j >= a.v) continue;
          float x = static_cast<float>(row[e + j]);
          if (bits >> j & 1) x = __uint_as_float(table[g * P + j]);
          else if (kBias >= 0) x += ld_any(a.bias, r * a.ldb + e + j, BT);
          if (forbidden<kMask>(a, r, e + j)) x = -__builtin_inff();
          orow[e + j] = static_cast<T>(x);
        }
      }
    }
    if (build) {
      __syncthreads();
      if (repeats > 0) {
        for (int i = lane; i < a.tile / 32; i += nt) owned[i] = 0;
        __syncthreads();
        for (int i = lane; i < repeats; i += nt) {
          const int at = places[i];
          words[i] = table[at], table[at] = 0;   // (0.f)
          atomicOr(&owned[at >> 5], 1u << (at & 31));
        }
        __syncthreads();
        sum_repeated(a, r, e0, table, owned);
        __syncthreads();
        const float rep = a.rep ? a.rep[r] : a.rep_s, pres = a.pres ? a.pres[r] : a.pres_s, freq = a.freq ? a.freq[r] : a.freq_s;
        for (int i = lane; i < repeats; i += nt) {
          const int at = places[i];
          const int64_t v = e0 + at;
          float x = adjust<kBias>(a, r, static_cast<int>(v), reinterpret_cast<float *>(list)[i], words[i],
                                  __uint_as_float(table[at]), rep, pres, freq);
          if (forbidden<kMask>(a, r, v)) x = -__builtin_inff();
          orow[v] = static_cast<T>(x);
        }
        __syncthreads();
      }
    }
  }
}

template <int DT, int kBias>
void launch_logits(const LogitsArgs &a, dim3 grid, dim3 block, size_t lds, hipStream_t s) {
  if (a.mask_kind == SBOD_MASK_BITS) hipLaunchKernelGGL((k_logits<DT, SBOD_MASK_BITS, kBias>), grid, block, lds, s, a);
  else if (a.mask_kind == SBOD_MASK_BYTES) hipLaunchKernelGGL((k_logits<DT, SBOD_MASK_BYTES, kBias>), grid, block, lds, s, a);
  else hipLaunchKernelGGL((k_logits<DT, SBOD_MASK_NONE, kBias>), grid, block, lds, s, a);
}
template <int DT>
void launch_logits(const LogitsArgs &a, dim3 grid, dim3 block, size_t lds, hipStream_t s) {
  if (!a.bias) launch_logits<DT, -1>(a, grid, block, lds, s);
  else if (a.bias_dt == SBOD_DT_F32) launch_logits<DT, SBOD_DT_F32>(a, grid, block, lds, s);
  else launch_logits<DT, DT>(a, grid, block, lds, s);
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
  SBOD_REQUIRE(known_dt(dtype) && (!bias || bias_dtype == SBOD_DT_F32 || bias_dtype == dtype), "sbod_logits_process: dtype %d / %d", dtype, bias_dtype);
  SBOD_REQUIRE(n >= 0 && v >= 1 && v < (1ll << 31) - 65536 && ld >= v && out_ld >= v && n < (1ll << 40) / v,
               "sbod_logits_process: logits [%lld, %lld], row strides %lld / %lld", static_cast<long long>(n),
               static_cast<long long>(v), static_cast<long long>(ld), static_cast<long long>(out_ld));
  SBOD_REQUIRE(history_cols >= 0 && history_cols <= kCount && bias_cols >= 0 && bias_cols <= kMaxBiases && history_ld >= 0 && bias_ld >= 0 &&
                   bias_ids_ld >= 0 && bias_values_ld >= 0 && mask_ld >= 0,
               "sbod_logits_process: %lld history entries, %d listed biases (0 .. %u, 0 .. %d), or a negative stride",
               static_cast<long long>(history_cols), bias_cols, kCount, kMaxBiases);
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
  // a row's labels from the 16-byte boundary below it on
  const bool even = (reinterpret_cast<uintptr_t>(logits) | ld * elt_bytes(dtype)) % 16 == 0;
  const int64_t most = even ? v : v + 16 / static_cast<int64_t>(elt_bytes(dtype)) - 1;
  a.ntile = static_cast<int>((most + kLogTile - 1) / kLogTile);
  a.tile = static_cast<int>(most < kLogTile ? (most + 31) / 32 * 32 : kLogTile);
  // threads for the tile's granules, two (four of float32) each
  const dim3 block(a.tile <= 1024 ? 128 : a.tile <= kLogTile / 2 ? 256 : kLogThreads);
  const int64_t items = n * a.ntile;
  const dim3 grid(static_cast<unsigned>(items < 65536 ? items : 65536));
  const size_t lds = a.len > 0 || a.m > 0 ? a.tile * sizeof(uint32_t) + list_size(a.tile, a.m) * sizeof(uint16_t) + a.tile / 4 +
                                                a.m / 2 * (sizeof(uint32_t) + sizeof(uint16_t))
                                          : 0;   // (62 KB at most)
  hipStream_t s = as_stream(stream);
  if (dtype == SBOD_DT_F32) launch_logits<SBOD_DT_F32>(a, grid, block, lds, s);
  else if (dtype == SBOD_DT_BF16) launch_logits<SBOD_DT_BF16>(a, grid, block, lds, s);
  else launch_logits<SBOD_DT_F16>(a, grid, block, lds, s);
  SBOD_LAUNCHED("k_logits");
  return SBOD_OK;
}
