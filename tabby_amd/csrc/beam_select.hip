// Beam search's selection: the best continuations of each group of beams.
//
// For group g, beam b and token t allowed in that beam's row x of logits:
//   score(b, t) = s[g, b] + (x_t - log sum_{u allowed} exp(x_u));
// an ended beam has one continuation, the padding token at its own score s[g, b]. The group's first
// `count` by score are kept, equal scores in the order of (b, t).
//
// Two kernels. The first reads the logits and leaves, for each row, its largest logit M, the sum S of
// exp(x - M), and its first `count` entries by (logit, index) -- adding s and subtracting the row's
// logarithm keeps their order, so no entry after those can be among the group's. The second adds M,
// log S and s to each group's entries and takes the best. Sums and scores are in 64 bits: whether
// a continuation of one beam comes before another beam's hangs on the difference of two logarithms.

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
constexpr int kEntriesMax = kBeamsMax * kCountMax;  // a group's entries, all of them in LDS
constexpr int kRowWaves = 16;
constexpr int kRowBlock = kRowWaves * 64;
constexpr int kMergeWaves = 16;
constexpr int kMergeBlock = kMergeWaves * 64;

// What the first kernel leaves of a row, beside its entries.
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
  int pad_id;
  int32_t *tokens, *parents;
  float *out_scores;
  int32_t *status;
  RowSum *sums;       // [rows]
  uint64_t *entries;  // [rows][count]
};

// A beam that has continuations in the vocabulary.
__device__ __forceinline__ bool beam_reads(const BeamArgs &a, int row) {
  return a.scores[row] > -INFINITY && !(a.done && a.done[row]);
}

template <int DT>
__global__ __launch_bounds__(kRowBlock) void beam_row_kernel(BeamArgs a) {
  using E = Elem<DT>;
  __shared__ BlockScratchT<kRowWaves> scratch;
  __shared__ uint32_t hist[kBins];
  __shared__ uint64_t top[kCountMax];
  __shared__ uint32_t taken;
  const int row = (int)blockIdx.x;
  if (!beam_reads(a, row)) {
    if (threadIdx.x == 0) a.sums[row] = RowSum{0.0, -INFINITY, 0, 0, 0};
    return;
  }
  const auto *src = (const typename E::Bits *)a.logits + (int64_t)row * a.row_stride;
  const uint32_t *mask = a.allowed ? a.allowed + (int64_t)row * a.words : nullptr;
  auto for_each = [&](auto f) {
    for (int t = (int)threadIdx.x; t < a.vocab; t += kRowBlock) {
      if (mask && !((mask[t >> 5] >> (t & 31)) & 1u)) continue;
      f(E::widen(src[t]), t);
    }
  };
  float m = -INFINITY;
  uint32_t valid = 0, bad = 0;
  for_each([&](float x, int) {
    if (x > -INFINITY) ++valid;
    if (!(x < INFINITY)) bad = 1;
    m = fmaxf(m, x);
  });
  m = value_of(wave_max_u32(key_of(m)));
  __syncthreads();
  if (lane_id() == 0) scratch.f[wave_id()] = m;
  uint32_t n, anybad;
  block_exclusive_scan(valid, scratch, &n);
  block_exclusive_scan(bad, scratch, &anybad);
  for (int i = 0; i < kRowWaves; ++i) m = fmaxf(m, scratch.f[i]);
  if (anybad || n == 0) {
    if (threadIdx.x == 0) a.sums[row] = RowSum{0.0, -INFINITY, 0, anybad ? 1 : 0, 0};
    return;
  }
  double sum = 0.0;
  for_each([&](float x, int) { sum += exp((double)x - (double)m); });
  sum = block_sum(sum, scratch);
  const uint32_t need = min(n, (uint32_t)a.count);
  auto composites = [&](auto f) {
    for_each([&](float x, int t) {
      if (x > -INFINITY) f(composite(key_of(x), (uint32_t)t));
    });
  };
  const SelectResult r = radix_select(composites, need, hist, scratch);
  if (threadIdx.x == 0) taken = 0;
  if (threadIdx.x < kCountMax) top[threadIdx.x] = 0;
  __syncthreads();
  composites([&](uint64_t c) {
    if (selected(c, r)) top[atomicAdd(&taken, 1u)] = c;
  });
  __syncthreads();
  bitonic_sort_desc<kRowWaves>(top, next_pow2((int)need));
  for (int i = (int)threadIdx.x; i < (int)need; i += kRowBlock) a.entries[(int64_t)row * a.count + i] = top[i];
  if (threadIdx.x == 0) a.sums[row] = RowSum{sum, m, (int)need, 0, 0};
}

// Order-preserving 64-bit key of a score that is no NaN.
__device__ __forceinline__ uint64_t score_key(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double score_of(uint64_t k) {
  return __longlong_as_double((long long)(k ^ (~(uint64_t)((int64_t)k >> 63) | 0x8000000000000000ull)));
}

__global__ __launch_bounds__(kMergeBlock) void beam_merge_kernel(BeamArgs a) {
  __shared__ BlockScratchT<kMergeWaves> scratch;
  __shared__ uint32_t hist[kBins];
  __shared__ uint64_t keys[kEntriesMax];  // scores
  __shared__ uint64_t tags[kEntriesMax];  // beam << 32 | token: the order of equal scores
  __shared__ uint16_t kept[kEntriesMax];  // the entries that the ranking looks at
  __shared__ double base[kBeamsMax], norm[kBeamsMax];
  __shared__ uint32_t total, left, bad;
  const int g = (int)blockIdx.x, t = (int)threadIdx.x;
  const int row0 = g * a.beams;
  if (t == 0) total = left = bad = 0;
  __syncthreads();
  if (t < a.beams) {
    const int row = row0 + t;
    const float s = a.scores[row];
    const RowSum rs = a.sums[row];
    if (!(s < INFINITY) || rs.bad) atomicOr(&bad, 1u);
    base[t] = (double)s;
    norm[t] = rs.count > 0 ? (double)rs.max + log(rs.sum) : 0.0;
    if (a.done && a.done[row] && s > -INFINITY) {
      const uint32_t at = atomicAdd(&total, 1u);
      keys[at] = score_key((double)s);
      tags[at] = ((uint64_t)t << 32) | (uint32_t)a.pad_id;
    }
  }
  __syncthreads();
  for (int i = t; i < a.beams * a.count; i += kMergeBlock) {
    const int b = i / a.count, j = i - b * a.count;
    if (j >= a.sums[row0 + b].count) continue;
    const uint64_t c = a.entries[(int64_t)(row0 + b) * a.count + j];
    const uint32_t at = atomicAdd(&total, 1u);
    keys[at] = score_key(base[b] + ((double)value_of(composite_key(c)) - norm[b]));
    tags[at] = ((uint64_t)b << 32) | composite_index(c);
  }
  __syncthreads();
  const uint32_t n = bad ? 0u : total;
  const uint32_t need = min(n, (uint32_t)a.count);
  if (need > 0) {
    const SelectResult r = radix_select(
        [&](auto f) {
          for (uint32_t i = t; i < n; i += kMergeBlock) f(keys[i]);
        },
        need, hist, scratch);
    for (uint32_t i = t; i < n; i += kMergeBlock)
      if (selected(keys[i], r)) kept[atomicAdd(&left, 1u)] = (uint16_t)i;
    __syncthreads();
    for (uint32_t i = t; i < left; i += kMergeBlock) {
      const uint64_t key = keys[kept[i]], tag = tags[kept[i]];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < left; ++j) {
        const uint64_t k = keys[kept[j]];
        rank += (k > key || (k == key && tags[kept[j]] < tag)) ? 1u : 0u;
      }
      if (rank < need) {
        const int64_t o = (int64_t)g * a.count + rank;
        a.tokens[o] = (int32_t)(uint32_t)tag;
        a.parents[o] = (int32_t)(tag >> 32);
        a.out_scores[o] = (float)score_of(key);
      }
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
  if ((int64_t)groups * beams > INT32_MAX) return record_failure(TABBY_EINVAL, "groups x beams must fit 32 bits");
  return TABBY_OK;
}

int64_t sums_bytes(int64_t rows) { return (rows * (int64_t)sizeof(RowSum) + 15) / 16 * 16; }

template <int DT>
int launch_rows(const BeamArgs &a, hipStream_t s) {
  hipLaunchKernelGGL(beam_row_kernel<DT>, dim3((unsigned)(a.groups * a.beams)), dim3(kRowBlock), 0, s, a);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

}  // namespace
}  // namespace tabby

using namespace tabby;

extern "C" int tabby_beam_workspace(int32_t groups, int32_t beams, int32_t vocab, int32_t count, int64_t *bytes) {
  if (!bytes) return record_failure(TABBY_EINVAL, "null pointer");
  const int rc = check_beam_shape(groups, beams, vocab, count);
  if (rc) return rc;
  const int64_t rows = (int64_t)groups * beams;
  *bytes = sums_bytes(rows) + rows * count * (int64_t)sizeof(uint64_t);
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
  BeamArgs a{logits_dev, row_stride, scores_dev, allowed_dev, done_dev, groups, beams, vocab, count,
             (vocab - 1) / 32 + 1, pad_id, tokens_dev, parents_dev, out_scores_dev, status_dev,
             (RowSum *)workspace_dev, (uint64_t *)((char *)workspace_dev + sums_bytes(rows))};
  const hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case TABBY_F32: rc = launch_rows<TABBY_F32>(a, s); break;
    case TABBY_F16: rc = launch_rows<TABBY_F16>(a, s); break;
    default: rc = launch_rows<TABBY_BF16>(a, s); break;
  }
  if (rc) return rc;
  hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)groups), dim3(kMergeBlock), 0, s, a);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}
