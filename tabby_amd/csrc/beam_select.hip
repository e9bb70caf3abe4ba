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
// can be among the group's (where rounding makes scores of one beam equal that its logits tell apart, the logits
// have decided). The second adds M, log S and s to each group's entries and takes the
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
#include "row_scan.h"

namespace tabby {
namespace {

constexpr int kBeamsMax = 64;
constexpr int kCountMax = 128;
constexpr int kPartsMax = 32;
constexpr int kRowsMax = (1 << 23) - 1;       // of 512 threads each
constexpr int kEntriesMax = 8192;             // a group's entries, all of them in LDS
static_assert(kBeamsMax * kCountMax <= kEntriesMax, "a group's entries");
static_assert(kCountMax == kListCountMax, "what a list keeps");

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

// One workgroup of NW waves to a part of a row, every element read once. Many rows are bound by the issue of
// the 64-bit terms (16 operations an element) and by HBM, which one wave does not overlap: it asks for its next
// chunk before it looks at this one, but waits for it at the loop's end, and the unit's other waves cover that.
// 512 rows of 151,936 f32 in 65 us, 4.8 TB/s; the whole call 67, from f16 63, from bf16 59. Few rows are bound by
// latency: the load, the bound, the list, the ranks (four rows in 19 parts each: 7.7 us).
template <int DT, bool MASK, int NW>
__global__ __launch_bounds__(NW * 64) void beam_row_kernel(BeamArgs a) {
  using Reader = PartReader<DT, MASK>;
  constexpr int kBlockN = NW * 64;
  __shared__ ListScratch<NW> scratch;
  __shared__ double wave_sum_[NW];
  __shared__ float wave_ref[NW], wave_max_[NW];
  const int row = (int)blockIdx.x / a.parts, part = (int)blockIdx.x - row * a.parts;
  const int t = (int)threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int begin = part * a.part_len, len = min(a.part_len, a.vocab - begin);
  const uint32_t *const mask = a.allowed ? a.allowed + (int64_t)row * a.words : nullptr;
  const Reader reader((const typename Reader::Bits *)a.logits + (int64_t)row * a.row_stride, MASK ? mask : nullptr, a.words, begin, len);
  typename Reader::Raw raw, next;
  float x[kLane];
  int c = wave;
  reader.load(c, raw);
  reader.load(c + NW, next);
  asm volatile("" ::: "memory");  // on their way before the row's state is asked for
  if (!beam_reads(a, row)) {
    if (t == 0) a.sums[blockIdx.x] = RowSum{0.0, -INFINITY, 0, 0, 0};
    return;
  }
  float top;  // of the lane's elements of the chunk; NaN if one of them is
  if (c < reader.chunks) {
    reader.widen(raw, c, x);
    top = chunk_max(x);
  } else {
#pragma unroll
    for (int i = 0; i < kLane; ++i) x[i] = -INFINITY;
    top = -INFINITY;
  }
  RowList<NW> list(scratch, a.count, wave, top);

  double sum = 0.0;
  float ref = -INFINITY, largest = -INFINITY;  // terms are exp(x - ref)
  auto take = [&]() {
    list.take(reader, c, x, top);
    if (__ballot(top - ref > 600.0f)) {
      // The first chunk with an element, or one far above: another reference. (The difference is rounded near 600
      // only; ref + 600 would be 1,024 above a ref of 2^33.)
      const float m = wave_max(top);
      if (m < INFINITY) {
        sum *= exp_or_none<false>((double)ref - (double)m);
        ref = m;
      }
    }
    largest = fmaxf(largest, top);
    // A chunk whose terms are all below e^-50 is left out: it would add 2e-22 an element to a sum of at least one,
    // 3e-17 over 151,936 and 5e-14 over the longest row, less than the terms' own error. Masks that leave little
    // cost no exponentials.
    if (__ballot(top >= ref - 50.0f) && ref > -INFINITY) {
      const double at = (double)ref;
      double part_sum[2] = {0.0, 0.0};
#pragma unroll
      for (int i = 0; i < kLane; ++i) part_sum[i & 1] += exp_or_none<false>((double)x[i] - at);
      sum += part_sum[0] + part_sum[1];
    }
  };
  // Two of these workgroups share a unit, and its waves issue the oldest first: the elder would end after 33 us
  // of 54 and leave the other alone with half the waves. Whoever is further along yields instead: the whole call of
  // 512 rows of 151,936 f32 74 -> 67 us, f16 68 -> 61.
  constexpr bool kYields = NW == 8;
  const int tenth = reader.chunks / 10, late[3] = {reader.chunks - tenth, reader.chunks - 3 * tenth, reader.chunks - 6 * tenth};
  if constexpr (kYields) __builtin_amdgcn_s_setprio(3);
  while (c < reader.chunks) {
    take();
    if constexpr (kYields) {
      if (c >= late[0]) __builtin_amdgcn_s_setprio(0);
      else if (c >= late[1]) __builtin_amdgcn_s_setprio(1);
      else if (c >= late[2]) __builtin_amdgcn_s_setprio(2);
    }
    c += NW;
    raw = next;
    if (c >= reader.chunks) break;
    reader.load(c + NW, next);
    const uint32_t shared = list.shared_bound();
    reader.widen(raw, c, x);
    top = chunk_max(x);
    list.theta = max(list.theta, shared);
  }
  largest = wave_max(largest);
  sum = wave_sum(sum);
  if (lane == 0) {
    wave_sum_[wave] = sum;
    wave_ref[wave] = ref;
    wave_max_[wave] = largest;
  }
  __syncthreads();
  const uint32_t n = list.pack();
  if (scratch.bad || n == 0) {
    if (t == 0) a.sums[blockIdx.x] = RowSum{0.0, -INFINITY, 0, scratch.bad ? 1 : 0, 0};
    return;
  }
  const uint32_t need = min(n, (uint32_t)a.count);
  if (wave == 0) {
    const float m = wave_max(lane < NW ? wave_max_[lane] : -INFINITY);
    double term = lane < NW ? wave_sum_[lane] : 0.0;
    if (term > 0.0) term *= exp_or_none<false>((double)wave_ref[lane] - (double)m);
    term = wave_sum(term);
    if (t == 0) a.sums[blockIdx.x] = RowSum{term, m, (int)need, 0, 0};
  }
  // A wave's share of the list that does not hold what lies at or above its bounds: from the row again.
  list.select(n, need, a.entries + (int64_t)blockIdx.x * a.count, [&](auto f) {
    for (int e = begin + t; e < begin + len; e += kBlockN) {
      if (mask && !((mask[e >> 5] >> (e & 31)) & 1u)) continue;
      const float v = Reader::E::widen(reader.row[e]);
      if (v > -INFINITY) f(composite(key_of(v), (uint32_t)e));
    }
  });
}

// Order-preserving 64-bit key of a score that is no NaN.
__device__ __forceinline__ uint64_t score_key(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double score_of(uint64_t k) {
  return __longlong_as_double((long long)(k ^ (~(uint64_t)((int64_t)k >> 63) | 0x8000000000000000ull)));
}

// One workgroup of NW waves to a group of at most NW * 64 * EACH entries and NW * 64 parts: its beams' entries
// become scores, those that may be among the best `count` go to LDS, and there each is ranked by counting
// those that come before it. Bound by the latency of its few steps.
template <int NW, int EACH>
__global__ __launch_bounds__(NW * 64) void beam_merge_kernel(BeamArgs a, int width) {
  constexpr int kBlockN = NW * 64;
  constexpr int kHeld = kBlockN * EACH;
  __shared__ uint64_t keys[kHeld];  // scores
  __shared__ uint64_t tags[kHeld];  // beam << 32 | token: the order of equal scores
  __shared__ int32_t part_count[kBlockN];
  __shared__ double base[kBeamsMax], norm[kBeamsMax];
  __shared__ BoundScratch<NW> bounds;
  __shared__ uint32_t held, bad;
  const int g = (int)blockIdx.x, t = (int)threadIdx.x, lane = t & 63;
  const int row0 = g * a.beams;
  const int slots = a.beams * a.parts * a.count;
  const uint64_t *entries = a.entries + (int64_t)row0 * a.parts * a.count;
  // A lane holds its entries, or reads them twice where there are many.
  constexpr bool kHolds = EACH <= 4;
  uint64_t entry[kHolds ? EACH : 1];
  if constexpr (kHolds) {
#pragma unroll
    for (int j = 0; j < EACH; ++j) entry[j] = j * kBlockN + t < slots ? entries[j * kBlockN + t] : 0;
  }
  // `width` neighbouring lanes to a beam, a power of two up to kPartsMax, one to a part.
  const int beam = t / width, part = t & (width - 1);
  RowSum rs{0.0, -INFINITY, 0, 0, 0};
  float score = 0.0f;
  int ended = 0;
  if (beam < a.beams) {
    if (part < a.parts) rs = a.sums[(int64_t)(row0 + beam) * a.parts + part];
    score = a.scores[row0 + beam];
    ended = a.done ? a.done[row0 + beam] : 0;
  }
  if (t == 0) held = bad = 0;
  if (beam < a.beams && part < a.parts) part_count[beam * a.parts + part] = rs.count;
  float m = rs.max;
#pragma unroll
  for (int stride = 1; stride < kPartsMax; stride *= 2)
    if (stride < width) m = fmaxf(m, xor_lane_by(m, stride));
  double sum = rs.count > 0 ? rs.sum * exp_or_none<false>((double)rs.max - (double)m) : 0.0;
#pragma unroll
  for (int stride = 1; stride < kPartsMax; stride *= 2)
    if (stride < width) sum += xor_lane_by(sum, stride);
  const bool leads = beam < a.beams && part == 0;
  const bool stays = leads && ended && score > -INFINITY;  // as it is: one continuation
  if (leads) {
    base[beam] = (double)score;
    norm[beam] = m > -INFINITY ? (double)m + log(sum) : 0.0;
  }
  __syncthreads();
  if (rs.bad || !(score < INFINITY)) bad = 1;
  // Scores; 0 is below every one.
  const float per_list = 1.0f / (float)a.count, per_beam = 1.0f / (float)(a.count * a.parts);  // i + 1/2 < 2^13 has bits to spare
  auto beam_of = [&](int i) { return (int)(((float)i + 0.5f) * per_beam); };
  auto key_at = [&](int i, uint64_t e) -> uint64_t {
    if (i >= slots) return 0;
    const int l = (int)(((float)i + 0.5f) * per_list), b = beam_of(i);
    if (i - l * a.count >= part_count[l]) return 0;
    return score_key(base[b] + ((double)value_of(composite_key(e)) - norm[b]));
  };
  uint64_t key[kHolds ? EACH : 1];
  uint64_t best = stays ? score_key((double)score) : 0;
  if constexpr (kHolds) {
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      key[j] = key_at(j * kBlockN + t, entry[j]);
      best = max(best, key[j]);
    }
  } else {
#pragma unroll 1
    for (int i = t; i < slots; i += kBlockN) best = max(best, key_at(i, entries[i]));
  }
  // A bound by the upper half of the keys, where it saves more than it takes.
  uint32_t theta = 0;
  if (slots > kBlockN / 4) theta = bound_of<NW>((uint32_t)(best >> 32), a.count, bounds);
  auto keep = [&](uint64_t k, auto tag) {
    const bool in = k != 0 && (uint32_t)(k >> 32) >= theta;
    const uint64_t who = __ballot(in);
    if (!who) return;
    uint32_t at = 0;
    if (lane == 0) at = atomicAdd(&held, (uint32_t)__popcll(who));
    at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
    if (in) {
      at += lanes_before(who);
      keys[at] = k;
      tags[at] = tag();
    }
  };
  auto tag_at = [&](int i, uint64_t e) { return ((uint64_t)beam_of(i) << 32) | composite_index(e); };
  if constexpr (kHolds) {
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      if (j * kBlockN >= slots) break;
      keep(key[j], [&] { return tag_at(j * kBlockN + t, entry[j]); });
    }
  } else {
#pragma unroll 1
    for (int i = t; i - t < slots; i += kBlockN) {
      const uint64_t e = i < slots ? entries[i] : 0;
      keep(key_at(i, e), [&] { return tag_at(i, e); });
    }
  }
  if (a.done) keep(stays ? score_key((double)score) : 0, [&] { return ((uint64_t)beam << 32) | (uint32_t)a.pad_id; });
  __syncthreads();
  const uint32_t n = bad ? 0u : held;
  const uint32_t need = min(n, (uint32_t)a.count);
  const int share = share_of(kBlockN, n);
  for (uint32_t i = (uint32_t)t / share; i < (n + kBlockN - 1) / kBlockN * kBlockN / share; i += kBlockN / share) {
    const uint64_t k = i < n ? keys[i] : 0, tg = i < n ? tags[i] : 0;
    const uint32_t rank = rank_of(share, n, [&](uint32_t j) { return keys[j] > k || (keys[j] == k && tags[j] < tg); });
    if (i < n && rank < need && (t & (share - 1)) == 0) {
      const int64_t o = (int64_t)g * a.count + rank;
      a.tokens[o] = (int32_t)(uint32_t)tg;
      a.parents[o] = (int32_t)(tg >> 32);
      a.out_scores[o] = (float)score_of(k);
    }
  }
  for (int i = (int)need + t; i < a.count; i += kBlockN) {
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
  if ((int64_t)groups * beams > kRowsMax)
    return record_failure(TABBY_EINVAL, "groups x beams must be at most " + std::to_string(kRowsMax) + ": a launch's threads must fit 32 bits");
  return TABBY_OK;
}

int64_t sums_bytes(int64_t lists) { return (lists * (int64_t)sizeof(RowSum) + 15) / 16 * 16; }

constexpr int kCus = 256;          // an MI355X's compute units
constexpr int kPartMin = 8192;     // a chunk to each of eight waves

// Few rows are cut into parts, a workgroup each, until there is about one to a compute unit; a group's
// entries have to fit its merge. (Its parts do: they are at most kCus.)
int beam_parts(int64_t rows, int beams, int vocab, int count) {
  int64_t parts = std::min<int64_t>({kCus / std::max<int64_t>(rows, 1), (vocab + kPartMin - 1) / kPartMin, kPartsMax});
  parts = std::min<int64_t>(parts, kEntriesMax / (beams * count));
  return (int)std::max<int64_t>(parts, 1);
}

template <int DT, bool MASK, int NW>
int launch_block(const BeamArgs &a, unsigned blocks, hipStream_t s) {
  hipLaunchKernelGGL((beam_row_kernel<DT, MASK, NW>), dim3(blocks), dim3(NW * 64), 0, s, a);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

template <int DT, bool MASK>
int launch_rows(const BeamArgs &a, hipStream_t s) {
  const int64_t blocks = (int64_t)a.groups * a.beams * a.parts;
  // Four or eight waves where they have a chunk each. Else, up to a workgroup for each compute unit: sixteen;
  // more: eight, two to a unit at once.
  if (a.part_len <= 4 * kChunk) return launch_block<DT, MASK, 4>(a, (unsigned)blocks, s);
  if (blocks <= kCus && a.part_len > 8 * kChunk) return launch_block<DT, MASK, 16>(a, (unsigned)blocks, s);
  return launch_block<DT, MASK, 8>(a, (unsigned)blocks, s);
}

template <int NW, int EACH>
int launch_merge(const BeamArgs &a, int width, hipStream_t s) {
  hipLaunchKernelGGL((beam_merge_kernel<NW, EACH>), dim3((unsigned)a.groups), dim3(NW * 64), 0, s, a, width);
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
  // Parts begin on a word of the mask.
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
  int width = 1;
  while (width < parts) width *= 2;
  // As few waves, and as little code, as hold the entries: a launch runs most of it once.
  const int slots = beams * parts * count;
  if (beams * width <= 256 && slots <= 256) return launch_merge<4, 1>(a, width, s);
  if (beams * width <= 256 && slots <= 1024) return launch_merge<4, 4>(a, width, s);
  return slots <= 4096 ? launch_merge<16, 4>(a, width, s) : launch_merge<16, 8>(a, width, s);
}
