// Beam search's selection: the best continuations of each group of beams.
//
// For group g, beam b and token t allowed in that beam's row x of logits:
//   score(b, t) = s[g, b] + (x_t - log sum_{u allowed} exp(x_u));
// an ended beam has one continuation, the padding token at its own score s[g, b]. The group's first
// `count` by score are kept, equal scores in the order of (b, t).
//
// Two kernels. The first reads the logits and leaves, for each row (or each part of one, where rows
// are few), its largest logit M, the sum S of exp(x - M), and its first `count` entries by (logit,
// index) -- adding s and subtracting the row's logarithm keeps their order, so no entry after those
// can be among the group's. The second adds M, log S and s to each group's entries and takes the
// best. Sums and scores are in 64 bits: whether a continuation of one beam comes before another
// beam's hangs on the difference of two logarithms.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "abi_internal.h"
#include "block_ops.h"
#include "device_math.h"
#include "elem.h"

namespace tabby {
namespace {

constexpr int kBeamsMax = 64;
constexpr int kCountMax = 128;
constexpr int kPartsMax = 16;
constexpr int kVocabMax = 1 << 28;            // a part's bytes fit a buffer resource
constexpr int kEntriesMax = 8192;             // a group's entries, all of them in LDS
constexpr int kChunk = 1024;                  // elements a wave takes at a time
constexpr int kLane = kChunk / 64;            // of them to a lane
constexpr int kListMax = 2048;                // entries above the bound that LDS holds
constexpr int kMergeWaves = 16;
constexpr int kMergeBlock = kMergeWaves * 64;
static_assert(kBeamsMax * kCountMax <= kEntriesMax && kBeamsMax * kPartsMax <= kMergeBlock, "a group's entries and sums");

// What the first kernel leaves of a row's part, beside its entries.
struct RowSum {
  double sum;     // of exp(x - max)
  float max;
  int32_t count;  // entries written
  int32_t bad;    // a NaN or +inf where the row may look
  int32_t reserved;
};

struct BeamArgs {
  const void *logits;
  int64_t row_stride;
  const float *scores;
  const uint32_t *allowed;  // [rows][words] or null
  const int32_t *done;      // [rows] or null
  int groups, beams, vocab, count, words;
  int parts, part_len;
  int pad_id;
  int32_t *tokens, *parents;
  float *out_scores;
  int32_t *status;
  RowSum *sums;       // [rows][parts]
  uint64_t *entries;  // [rows][parts][count]
};

// A beam that has continuations in the vocabulary.
__device__ __forceinline__ bool beam_reads(const BeamArgs &a, int row) {
  return a.scores[row] > -INFINITY && !(a.done && a.done[row]);
}

// 2^t in 64 bits for t in [-1000, 1000]: the nearest whole power by adding and taking away 1.5 * 2^52,
// whose low word then holds it, and for the rest f in [-1/2, 1/2] the polynomial of degree 7 through
// 2^f at the Chebyshev nodes, within 5e-11 of it. A sum of such terms decides the order of two
// beams' continuations only where their scores are that close.
__device__ __forceinline__ double exp2_64(double t) {
  const double magic = 6755399441055744.0;
  const double shifted = t + magic;
  const double f = t - (shifted - magic);
  double p = 1.530370102315244e-05;
  p = __builtin_fma(p, f, 0.0001546972921563772);
  p = __builtin_fma(p, f, 0.0013333478472326247);
  p = __builtin_fma(p, f, 0.009618025613309008);
  p = __builtin_fma(p, f, 0.055504109063275894);
  p = __builtin_fma(p, f, 0.24022651213498245);
  p = __builtin_fma(p, f, 0.6931471805568318);
  p = __builtin_fma(p, f, 0.9999999999595618);
  const uint32_t n = (uint32_t)__double_as_longlong(shifted);
  const uint64_t bits = (uint64_t)__double_as_longlong(p);
  return __longlong_as_double((long long)(((uint64_t)((uint32_t)(bits >> 32) + (n << 20)) << 32) | (uint32_t)bits));
}

constexpr double kLog2e = 1.4426950408889634;

// The larger of two, NaN if either is: a chunk's maximum shows that it holds a NaN.
__device__ __forceinline__ float max_or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// One part of one row, read through 16-byte loads from the boundary at or before its start:
// position p of the part is element begin + p - lead. What lies before the part or after it is set to
// -inf where the first or the last chunk is taken apart, and the buffer's range ends with the last
// 16 bytes that hold an element.
template <int DT, bool MASK>
struct PartReader {
  using E = Elem<DT>;
  static constexpr int kLoads = kLane / E::kVec;
  static constexpr int kSize = (int)sizeof(typename E::Bits);
  struct Raw {
    u32x4 v[kLoads];
    uint32_t lo[MASK ? kLoads : 1], hi[MASK ? kLoads : 1];
  };
  RowBuffer buffer;
  const uint32_t *mask;
  int begin, len, lead, words, chunks;

  static __device__ __forceinline__ int lead_of(const typename E::Bits *at) { return (int)((uintptr_t)at % 16) / kSize; }

  __device__ __forceinline__ PartReader(const BeamArgs &a, int row, int begin_, int len_)
      : buffer(start(a, row, begin_) - lead_of(start(a, row, begin_)),
               (uint32_t)(((uint32_t)(lead_of(start(a, row, begin_)) + len_) * kSize + 15u) & ~15u)),
        mask(MASK ? a.allowed + (int64_t)row * a.words : nullptr),
        begin(begin_),
        len(len_),
        lead(lead_of(start(a, row, begin_))),
        words(a.words),
        chunks((lead + len_ + kChunk - 1) / kChunk) {}

  static __device__ __forceinline__ const typename E::Bits *start(const BeamArgs &a, int row, int begin) {
    return (const typename E::Bits *)a.logits + (int64_t)row * a.row_stride + begin;
  }

  // The position of the lane's first element of load u of chunk c.
  __device__ __forceinline__ int position(int c, int u) const {
    return c * kChunk + u * 64 * E::kVec + wave_lane() * E::kVec;
  }
  __device__ __forceinline__ int element(int c, int i) const {
    return begin - lead + position(c, i / E::kVec) + i % E::kVec;
  }

  // Past the last chunk it is the last one again, which nothing looks at.
  __device__ __forceinline__ void load(int c, Raw &r) const {
    c = min(c, chunks - 1);
    const uint32_t at = (uint32_t)wave_lane() * 16u;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) r.v[u] = buffer.load16(at, (uint32_t)c * (kChunk * kSize) + u * 1024u);
    if constexpr (MASK) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int w = (begin - lead + position(c, u)) >> 5;
        r.lo[u] = mask[min(max(w, 0), words - 1)];
        r.hi[u] = lead ? mask[min(max(w + 1, 0), words - 1)] : 0u;
      }
    }
  }

  __device__ __forceinline__ void widen(const Raw &r, int c, float (&x)[kLane]) const {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      float w[E::kVec];
      E::widen16(r.v[u], w);
#pragma unroll
      for (int j = 0; j < E::kVec; ++j) x[u * E::kVec + j] = w[j];
      if constexpr (MASK) {
        const uint32_t shift = (uint32_t)(begin - lead + position(c, u)) & 31u;
        const uint32_t bits = __builtin_amdgcn_alignbit(r.hi[u], r.lo[u], shift);
#pragma unroll
        for (int j = 0; j < E::kVec; ++j)
          x[u * E::kVec + j] = (bits >> j) & 1u ? x[u * E::kVec + j] : -INFINITY;
      }
    }
    if (c == 0 || c == chunks - 1) {
#pragma unroll
      for (int i = 0; i < kLane; ++i) {
        const int p = position(c, i / E::kVec) + i % E::kVec - lead;
        if (p < 0 || p >= len) x[i] = -INFINITY;
      }
    }
  }
};

// One workgroup of NW waves to a part of a row. HBM-bound: every element is read once.
template <int DT, bool MASK, int NW>
__global__ __launch_bounds__(NW * 64) void beam_row_kernel(BeamArgs a) {
  using Reader = PartReader<DT, MASK>;
  constexpr int kBlockN = NW * 64;
  __shared__ BlockScratchT<NW> scratch;
  __shared__ uint32_t hist[kBins];
  __shared__ uint64_t list[kListMax];
  __shared__ uint32_t first[NW * 64];  // the waves' largest lane maxima of their first chunks
  __shared__ uint32_t listed, bad, bound;
  __shared__ double wave_sum_[NW];
  __shared__ float wave_ref[NW], wave_max_[NW];
  const int row = (int)blockIdx.x / a.parts, part = (int)blockIdx.x - row * a.parts;
  const int t = (int)threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  if (!beam_reads(a, row)) {
    if (t == 0) a.sums[blockIdx.x] = RowSum{0.0, -INFINITY, 0, 0, 0};
    return;
  }
  const int begin = part * a.part_len, len = min(a.part_len, a.vocab - begin);
  const Reader reader(a, row, begin, len);
  if (t == 0) {
    listed = 0;
    bad = 0;
    bound = kNegInfKey + 1;
  }

  typename Reader::Raw raw;
  float x[kLane];
  int c = wave;
  reader.load(c, raw);
  auto chunk_max = [&]() {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < kLane; ++i) m = max_or_nan(m, x[i]);
    return m;
  };
  float top;  // of the lane's elements of the chunk; NaN if one of them is
  if (c < reader.chunks) {
    reader.widen(raw, c, x);
    top = chunk_max();
  } else {
#pragma unroll
    for (int i = 0; i < kLane; ++i) x[i] = -INFINITY;
    top = -INFINITY;
  }
  // The first bound: each wave offers the largest of its lanes' maxima, 64 R of them in all, and the
  // count-th largest of those has `count` elements of the part at or above it.
  const int wide = a.count > 64 ? 4 : 2;
  const int offered = 64 * wide / NW;
  {
    uint32_t key[1] = {top == top ? key_of(top) : 0u};
    wave_sort_desc<1>(key);
    if (lane < offered) first[wave * offered + lane] = key[0];
  }
  __syncthreads();
  uint32_t theta;
  {
    uint32_t k;
    if (a.count > 64) {
      uint32_t v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = first[r * 64 + lane];
      wave_sort_desc<4>(v);
      k = a.count > 64 ? v[1] : v[0];
      k = (uint32_t)__builtin_amdgcn_readlane((int)k, (a.count - 1) & 63);
    } else {
      uint32_t v[2] = {first[lane], first[64 + lane]};
      wave_sort_desc<2>(v);
      k = (uint32_t)__builtin_amdgcn_readlane((int)v[0], a.count - 1);
    }
    theta = max(k, kNegInfKey + 1);
  }

  double sum = 0.0;
  float ref = 0.0f, rise = -INFINITY, largest = -INFINITY;  // terms are exp(x - ref); x > rise asks for another ref
  auto take = [&]() {
    // Elements at or above the bound join the list; a NaN is neither.
    float least = value_of(theta);
    if (__ballot(!(top < least))) {
      const uint32_t shared = *(volatile uint32_t *)&bound;
      if (shared > theta) theta = shared;
      if (__ballot(!(top < value_of(theta)))) {
        if (!(top < INFINITY)) bad = 1;
        if (a.count <= 64 && __popcll(__ballot(top >= value_of(theta))) > a.count) {
          // Many lanes have one: the count-th largest of the lanes' maxima is a better bound.
          uint32_t key[1] = {top == top ? key_of(top) : 0u};
          wave_sort_desc<1>(key);
          const uint32_t k = (uint32_t)__builtin_amdgcn_readlane((int)key[0], a.count - 1);
          if (k > theta) {
            theta = k;
            if (lane == 0) atomicMax(&bound, k);
          }
        }
        least = value_of(theta);
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < kLane; ++i) mine += x[i] >= least ? 1u : 0u;
        const uint32_t upto = wave_inclusive_scan_u32(mine);
        uint32_t at = 0;
        if (lane == 63) at = atomicAdd(&listed, upto);
        at = (uint32_t)__builtin_amdgcn_readlane((int)at, 63) + upto - mine;
#pragma unroll
        for (int i = 0; i < kLane; ++i) {
          if (x[i] >= least) {
            if (at < kListMax) list[at] = composite(key_of(x[i]), (uint32_t)reader.element(c, i));
            ++at;
          }
        }
      }
    }
    if (__ballot(top > rise)) {
      // The first chunk with an element, or one far above: another reference.
      const float m = wave_max(top);
      if (m < INFINITY) {
        sum *= exp2_64(fmax(((double)ref - (double)m) * kLog2e, -1000.0));
        ref = m;
        rise = m + 600.0f;
      }
    }
    largest = fmaxf(largest, top);
    if (rise > -INFINITY) {
      const double at = (double)ref;
      double part_sum[2] = {0.0, 0.0};
#pragma unroll
      for (int i = 0; i < kLane; ++i) part_sum[i & 1] += exp2_64(fmax(((double)x[i] - at) * kLog2e, -1000.0));
      sum += part_sum[0] + part_sum[1];
    }
  };
  typename Reader::Raw next;
  if (c < reader.chunks) {
    reader.load(c + NW, next);
    take();
    for (c += NW; c < reader.chunks; c += NW) {
      raw = next;
      reader.load(c + NW, next);
      reader.widen(raw, c, x);
      top = chunk_max();
      take();
    }
  }
  largest = wave_max(largest);
  sum = wave_sum(sum);
  if (lane == 0) {
    wave_sum_[wave] = sum;
    wave_ref[wave] = ref;
    wave_max_[wave] = largest;
  }
  __syncthreads();
  const uint32_t n = listed;
  if (bad || n == 0) {
    if (t == 0) a.sums[blockIdx.x] = RowSum{0.0, -INFINITY, 0, bad ? 1 : 0, 0};
    return;
  }
  const uint32_t need = min(n, (uint32_t)a.count);
  uint64_t *out = a.entries + (int64_t)blockIdx.x * a.count;
  if (t == 0) {
    float m = wave_max_[0];
    for (int w = 1; w < NW; ++w) m = fmaxf(m, wave_max_[w]);
    double s = 0.0;
    for (int w = 0; w < NW; ++w)
      if (wave_sum_[w] > 0.0) s += wave_sum_[w] * exp((double)wave_ref[w] - (double)m);
    a.sums[blockIdx.x] = RowSum{s, m, (int)need, 0, 0};
  }
  if (n <= (uint32_t)a.count) {
    for (uint32_t i = t; i < n; i += kBlockN) out[i] = list[i];
    return;
  }
  if (n <= (uint32_t)kBlockN) {
    if (t < (int)n) {
      const uint64_t v = list[t];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < n; ++j) rank += list[j] > v ? 1u : 0u;
      if (rank < need) out[rank] = v;
    }
    return;
  }
  auto pick = [&](auto for_each) {
    const SelectResult r = radix_select(for_each, need, hist, scratch);
    if (t == 0) scratch.slot = 0;
    __syncthreads();
    for_each([&](uint64_t v) {
      if (selected(v, r)) out[atomicAdd(&scratch.slot, 1u)] = v;
    });
  };
  if (n <= (uint32_t)kListMax) {
    pick([&](auto f) {
      for (uint32_t i = t; i < n; i += kBlockN) f(list[i]);
    });
  } else {
    // More than the list holds lie at or above every bound that the waves found: from the row again.
    const uint32_t *mask = a.allowed ? a.allowed + (int64_t)row * a.words : nullptr;
    const auto *src = Reader::start(a, row, 0);
    pick([&](auto f) {
      for (int e = begin + t; e < begin + len; e += kBlockN) {
        if (mask && !((mask[e >> 5] >> (e & 31)) & 1u)) continue;
        const float v = Reader::E::widen(src[e]);
        if (v > -INFINITY) f(composite(key_of(v), (uint32_t)e));
      }
    });
  }
}

// Order-preserving 64-bit key of a score that is no NaN.
__device__ __forceinline__ uint64_t score_key(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double score_of(uint64_t k) {
  return __longlong_as_double((long long)(k ^ (~(uint64_t)((int64_t)k >> 63) | 0x8000000000000000ull)));
}

// One workgroup to a group: its beams' entries become scores, and the best `count` are ranked by
// counting, for each, those that come before it. Bound by the latency of its few steps.
__global__ __launch_bounds__(kMergeBlock) void beam_merge_kernel(BeamArgs a) {
  __shared__ BlockScratchT<kMergeWaves> scratch;
  __shared__ uint32_t hist[kBins];
  __shared__ uint64_t keys[kEntriesMax];  // scores
  __shared__ uint64_t tags[kEntriesMax];  // beam << 32 | token: the order of equal scores
  __shared__ double space[kEntriesMax / 4];
  double *const part_sum = space;  // the parts' sums, maxima and counts
  float *const part_max = (float *)(space + kBeamsMax * kPartsMax);
  int32_t *const part_count = (int32_t *)(part_max + kBeamsMax * kPartsMax);
  uint16_t *const kept = (uint16_t *)space;  // once those are used up: the entries that are ranked
  __shared__ double base[kBeamsMax], norm[kBeamsMax];
  __shared__ uint32_t total, left, bad;
  const int g = (int)blockIdx.x, t = (int)threadIdx.x;
  const int row0 = g * a.beams;
  const int lists = a.beams * a.parts;
  if (t == 0) total = left = bad = 0;
  __syncthreads();
  if (t < lists) {
    const RowSum rs = a.sums[(int64_t)row0 * a.parts + t];
    part_sum[t] = rs.sum;
    part_max[t] = rs.max;
    part_count[t] = rs.count;
    if (rs.bad) bad = 1;
  }
  __syncthreads();
  if (t < a.beams) {
    const int row = row0 + t;
    const float s = a.scores[row];
    if (!(s < INFINITY)) bad = 1;
    float m = -INFINITY;
    for (int p = 0; p < a.parts; ++p) m = fmaxf(m, part_max[t * a.parts + p]);
    double sum = 0.0;
    for (int p = 0; p < a.parts; ++p)
      if (part_count[t * a.parts + p] > 0) sum += part_sum[t * a.parts + p] * exp((double)part_max[t * a.parts + p] - (double)m);
    base[t] = (double)s;
    norm[t] = m > -INFINITY ? (double)m + log(sum) : 0.0;
    if (a.done && a.done[row] && s > -INFINITY) {
      const uint32_t at = atomicAdd(&total, 1u);
      keys[at] = score_key((double)s);
      tags[at] = ((uint64_t)t << 32) | (uint32_t)a.pad_id;
    }
  }
  __syncthreads();
  for (int i = t; i < lists * a.count; i += kMergeBlock) {
    const int l = i / a.count, j = i - l * a.count;
    if (j >= part_count[l]) continue;
    const int b = l / a.parts;
    const uint64_t c = a.entries[(int64_t)row0 * a.parts * a.count + i];
    const uint32_t at = atomicAdd(&total, 1u);
    keys[at] = score_key(base[b] + ((double)value_of(composite_key(c)) - norm[b]));
    tags[at] = ((uint64_t)b << 32) | composite_index(c);
  }
  __syncthreads();
  const uint32_t n = bad ? 0u : total;
  const uint32_t need = min(n, (uint32_t)a.count);
  // More than a lane each: only those at or above the count-th score are ranked.
  const bool cut = n > (uint32_t)kMergeBlock;
  if (cut) {
    const SelectResult r = radix_select(
        [&](auto f) {
          for (uint32_t i = t; i < n; i += kMergeBlock) f(keys[i]);
        },
        need, hist, scratch);
    for (uint32_t i = t; i < n; i += kMergeBlock)
      if (selected(keys[i], r)) kept[atomicAdd(&left, 1u)] = (uint16_t)i;
    __syncthreads();
  }
  const uint32_t ranked = cut ? left : n;
  for (uint32_t i = t; i < ranked; i += kMergeBlock) {
    const uint32_t e = cut ? kept[i] : i;
    const uint64_t key = keys[e], tag = tags[e];
    uint32_t rank = 0;
    for (uint32_t j = 0; j < ranked; ++j) {
      const uint32_t o = cut ? kept[j] : j;
      const uint64_t k = keys[o];
      rank += (k > key || (k == key && tags[o] < tag)) ? 1u : 0u;
    }
    if (rank < need) {
      const int64_t o = (int64_t)g * a.count + rank;
      a.tokens[o] = (int32_t)(uint32_t)tag;
      a.parents[o] = (int32_t)(tag >> 32);
      a.out_scores[o] = (float)score_of(key);
    }
  }
  for (int i = (int)need + t; i < a.count; i += kMergeBlock) {
    const int64_t o = (int64_t)g * a.count + i;
    a.tokens[o] = -1;
    a.parents[o] = -1;
    a.out_scores[o] = -INFINITY;
  }
  if (t == 0 && a.status) a.status[g] = bad ? TABBY_EDOMAIN : n == 0 ? TABBY_EEMPTY : TABBY_OK;
}

int check_beam_shape(int32_t groups, int32_t beams, int32_t vocab, int32_t count) {
  if (groups < 1 || beams < 1 || vocab < 1) return record_failure(TABBY_EINVAL, "groups, beams and vocab must be >= 1");
  if (beams > kBeamsMax)
    return record_failure(TABBY_EINVAL, "beams must be between 1 and " + std::to_string(kBeamsMax) + ", got " + std::to_string(beams));
  if (count < 1 || count > kCountMax)
    return record_failure(TABBY_EINVAL, "count must be between 1 and " + std::to_string(kCountMax) + ", got " + std::to_string(count));
  if (vocab > kVocabMax) return record_failure(TABBY_EINVAL, "vocab must be at most " + std::to_string(kVocabMax));
  if ((int64_t)groups * beams > INT32_MAX / kPartsMax) return record_failure(TABBY_EINVAL, "groups x beams x " + std::to_string(kPartsMax) + " must fit 32 bits");
  return TABBY_OK;
}

int64_t sums_bytes(int64_t lists) { return (lists * (int64_t)sizeof(RowSum) + 15) / 16 * 16; }

constexpr int kCus = 256;          // an MI355X's compute units
constexpr int kPartMin = 16384;    // a part is worth a workgroup from here on

// Few rows are cut into parts, a workgroup each, until there is about one to a compute unit; a group's
// entries have to fit the merge's LDS.
int beam_parts(int64_t rows, int beams, int vocab, int count) {
  int64_t parts = std::min<int64_t>({kCus / std::max<int64_t>(rows, 1), vocab / kPartMin, kPartsMax});
  parts = std::min<int64_t>(parts, kEntriesMax / (beams * count));
  return (int)std::max<int64_t>(parts, 1);
}

template <int DT, bool MASK>
int launch_rows(const BeamArgs &a, hipStream_t s) {
  const int64_t blocks = (int64_t)a.groups * a.beams * a.parts;
  // Up to a workgroup for each compute unit: sixteen waves each; more: eight, two to a unit at once.
  if (blocks <= kCus) hipLaunchKernelGGL((beam_row_kernel<DT, MASK, 16>), dim3((unsigned)blocks), dim3(1024), 0, s, a);
  else hipLaunchKernelGGL((beam_row_kernel<DT, MASK, 8>), dim3((unsigned)blocks), dim3(512), 0, s, a);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

template <int DT>
int launch_type(const BeamArgs &a, hipStream_t s) {
  return a.allowed ? launch_rows<DT, true>(a, s) : launch_rows<DT, false>(a, s);
}

}  // namespace
}  // namespace tabby

using namespace tabby;

extern "C" int tabby_beam_workspace(int32_t groups, int32_t beams, int32_t vocab, int32_t count, int64_t *bytes) {
  if (!bytes) return record_failure(TABBY_EINVAL, "null pointer");
  const int rc = check_beam_shape(groups, beams, vocab, count);
  if (rc) return rc;
  // For these sizes and every smaller one: rows that are cut make at most kCus parts.
  const int64_t lists = std::max<int64_t>((int64_t)groups * beams, kCus);
  *bytes = sums_bytes(lists) + lists * count * (int64_t)sizeof(uint64_t);
  return TABBY_OK;
}

extern "C" int tabby_beam_select_device(const void *logits_dev, int32_t dtype, int64_t row_stride, int32_t groups,
                                        int32_t beams, int32_t vocab, const float *scores_dev,
                                        const uint32_t *allowed_dev, const int32_t *done_dev, int32_t pad_id,
                                        int32_t count, int32_t *tokens_dev, int32_t *parents_dev,
                                        float *out_scores_dev, int32_t *status_dev, void *workspace_dev,
                                        int64_t workspace_bytes, void *stream) {
  if (!logits_dev || !scores_dev || !tokens_dev || !parents_dev || !out_scores_dev || !workspace_dev)
    return record_failure(TABBY_EINVAL, "null pointer");
  int rc = check_beam_shape(groups, beams, vocab, count);
  if (rc) return rc;
  if (!known_dtype(dtype)) return record_failure(TABBY_EINVAL, "dtype must be TABBY_F32, TABBY_F16 or TABBY_BF16");
  if (groups * beams > 1 && row_stride < vocab) return record_failure(TABBY_EINVAL, "row_stride must be at least vocab");
  if ((uintptr_t)logits_dev % dtype_size(dtype) != 0)
    return record_failure(TABBY_EINVAL, "logits must be aligned to their elements");
  if (pad_id < 0) return record_failure(TABBY_EINVAL, "pad_id must be >= 0");
  int64_t need;
  rc = tabby_beam_workspace(groups, beams, vocab, count, &need);
  if (rc) return rc;
  if ((uintptr_t)workspace_dev % 16 != 0 || workspace_bytes < need)
    return record_failure(TABBY_EINVAL, "workspace must be 16-byte aligned and hold " + std::to_string(need) + " bytes");
  const int64_t rows = (int64_t)groups * beams;
  const int parts = beam_parts(rows, beams, vocab, count);
  // Parts begin on a mask word, and on 16 bytes where the row does.
  const int part_len = (int)((((int64_t)vocab + parts - 1) / parts + 31) / 32 * 32);
  BeamArgs a{logits_dev, row_stride, scores_dev, allowed_dev, done_dev, groups, beams, vocab, count,
             (vocab - 1) / 32 + 1, parts, part_len, pad_id, tokens_dev, parents_dev, out_scores_dev, status_dev,
             (RowSum *)workspace_dev, (uint64_t *)((char *)workspace_dev + sums_bytes(rows * parts))};
  const hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case TABBY_F32: rc = launch_type<TABBY_F32>(a, s); break;
    case TABBY_F16: rc = launch_type<TABBY_F16>(a, s); break;
    default: rc = launch_type<TABBY_BF16>(a, s); break;
  }
  if (rc) return rc;
  hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)groups), dim3(kMergeBlock), 0, s, a);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}
