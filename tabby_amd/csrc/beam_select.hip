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

namespace tabby {
namespace {

constexpr int kBeamsMax = 64;
constexpr int kCountMax = 128;
constexpr int kPartsMax = 32;
constexpr int kVocabMax = 1 << 28;            // places in a row in 32 bits, with room
constexpr int kRowsMax = (1 << 23) - 1;       // of 512 threads each
constexpr int kEntriesMax = 8192;             // a group's entries, all of them in LDS
constexpr int kChunk = 1024;                  // elements a wave takes at a time
constexpr int kLane = kChunk / 64;            // of them to a lane
constexpr int kListMax = 4096;                // entries above the bound that LDS holds, a share to each wave
static_assert(kBeamsMax * kCountMax <= kEntriesMax, "a group's entries");

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

typedef uint32_t uint32x2 __attribute__((ext_vector_type(2)));

// exp(d) in 64 bits for d in [-690, 690]: t = d log2(e) is split into the nearest whole number, found by adding
// and taking away 1.5 * 2^52, whose low word then holds it, and the rest f in [-1/2, 1/2]; for 2^f the
// polynomial of degree 7 through it at the Chebyshev nodes, within 5.5e-11 of it. A sum of such terms
// decides the order of two beams' continuations only where their scores are that close.
__device__ __forceinline__ double exp_64(double d) {
  constexpr double kLog2e = 1.4426950408889634;
  const double magic = 6755399441055744.0;
  const double shifted = __builtin_fma(d, kLog2e, magic);
  const double f = __builtin_fma(d, kLog2e, -(shifted - magic));
  double p = 1.530370102315244e-05;
  p = __builtin_fma(p, f, 0.0001546972921563772);
  p = __builtin_fma(p, f, 0.0013333478472326247);
  p = __builtin_fma(p, f, 0.009618025613309008);
  p = __builtin_fma(p, f, 0.055504109063275894);
  p = __builtin_fma(p, f, 0.24022651213498245);
  p = __builtin_fma(p, f, 0.6931471805568318);
  p = __builtin_fma(p, f, 0.9999999999595618);
  uint32x2 bits = __builtin_bit_cast(uint32x2, p);
  bits.y += __builtin_bit_cast(uint32x2, shifted).x << 20;
  return __builtin_bit_cast(double, bits);
}
// The same for any d <= 690, -inf too: below -690 nothing is left that a sum of at least 1 would hold. Above 690 the
// exponent's field runs over, and the result, NaN included, has nothing to do with exp.
__device__ __forceinline__ double exp_or_none(double d) { return exp_64(fmax(d, -690.0)); }

// The larger of two, NaN if either is: a chunk's maximum shows that it holds a NaN.
__device__ __forceinline__ float max_or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// One part of one row, 16 bytes to a lane from the part's first element on, wherever it lies (the hardware
// takes any address): which lane takes which element, and so the order of the sum, depends on its place in
// the row alone, and rows that are equal score alike to the last bit.
template <int DT, bool MASK>
struct PartReader {
  using E = Elem<DT>;
  using Bits = typename E::Bits;
  static constexpr int kLoads = kLane / E::kVec;
  static constexpr int kLoad = 64 * E::kVec;  // elements of a load
  struct Raw {
    u32x4 v[kLoads];
    uint32_t mask[MASK ? kLoads : 1];
  };
  const Bits *row;
  const uint32_t *mask;
  int begin, len, words, chunks;

  __device__ __forceinline__ PartReader(const BeamArgs &a, int r, int begin_, int len_)
      : row((const Bits *)a.logits + (int64_t)r * a.row_stride),
        mask(MASK ? a.allowed + (int64_t)r * a.words : nullptr),
        begin(begin_),
        len(len_),
        words(a.words),
        chunks((len_ + kChunk - 1) / kChunk) {}

  // The place in the part of the lane's first element of load u of chunk c.
  __device__ __forceinline__ int position(int c, int u) const { return c * kChunk + u * kLoad + wave_lane() * E::kVec; }
  __device__ __forceinline__ int element(int c, int i) const { return begin + position(c, i / E::kVec) + i % E::kVec; }

  // Past the last chunk it is the last one again, which nothing looks at.
  __device__ __forceinline__ void load(int c, Raw &r) const {
    c = min(c, chunks - 1);
    const Bits *from = row + begin + c * kChunk;
    const int lane = wave_lane() * E::kVec;
    if ((c + 1) * kChunk <= len) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) r.v[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(from + lane + u * kLoad));
    } else {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int left = len - position(c, u);
        r.v[u] = u32x4{0, 0, 0, 0};
        if (left >= E::kVec) {
          r.v[u] = *reinterpret_cast<const u32x4_any *>(from + lane + u * kLoad);
        } else {
#pragma unroll
          for (int j = 0; j < E::kVec - 1; ++j) {
            if (j < left) {
              const uint32_t b = from[lane + u * kLoad + j];
              if constexpr (E::kVec == 4) r.v[u][j] = b;
              else r.v[u][j / 2] |= b << (16 * (j & 1));
            }
          }
        }
      }
    }
    if constexpr (MASK) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) r.mask[u] = mask[min((begin + position(c, u)) >> 5, words - 1)];
    }
  }

  __device__ __forceinline__ void widen(const Raw &r, int c, float (&x)[kLane]) const {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      float w[E::kVec];
      E::widen16(r.v[u], w);
      uint32_t bits = 0;  // parts begin on a word of the mask, and a load lies within one
      if constexpr (MASK) bits = r.mask[u] >> ((uint32_t)position(c, u) & 31u);
#pragma unroll
      for (int j = 0; j < E::kVec; ++j) x[u * E::kVec + j] = !MASK || (bits >> j) & 1u ? w[j] : -INFINITY;
    }
    if (c == chunks - 1) {
#pragma unroll
      for (int i = 0; i < kLane; ++i)
        if (position(c, i / E::kVec) + i % E::kVec >= len) x[i] = -INFINITY;
    }
  }
};

// The k-th largest of the wave's 64 R values, k up to 64 (R = 1) or 128.
template <int R>
__device__ __forceinline__ uint32_t kth_largest(uint32_t (&v)[R], int k) {
  wave_sort_desc<R>(v);
  if constexpr (R == 1) return (uint32_t)__builtin_amdgcn_readlane((int)v[0], k - 1);
  else return (uint32_t)__builtin_amdgcn_readlane((int)(k > 64 ? v[1] : v[0]), (k - 1) & 63);
}

// The number of set lanes before this one.
__device__ __forceinline__ uint32_t lanes_before(uint64_t who) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
}

// A lower bound of the count-th largest of the keys that the workgroup's lanes hold, one each: the keys fall
// into 64 columns (256 where more than 32 are kept), and the count-th largest of the columns' largest has
// as many keys at or above it. Close to the count-th largest itself where the keys fall by chance; each
// wave's are turned by another angle so that an order among them matters less.
template <int NW>
struct BoundScratch {
  uint32_t keys[NW * 64];
  uint32_t bound;
};

template <int NW>
__device__ __forceinline__ uint32_t bound_of(uint32_t key, int count, BoundScratch<NW> &s) {
  const int lane = wave_lane(), wave = (int)threadIdx.x >> 6;
  s.keys[wave * 64 + ((lane + 5 * wave) & 63)] = key;
  __syncthreads();
  if (wave == 0) {
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) v[w & 3] = max(v[w & 3], s.keys[w * 64 + lane]);
    uint32_t all[1] = {max(max(v[0], v[1]), max(v[2], v[3]))};
    const uint32_t k = count <= 32 ? kth_largest<1>(all, count) : kth_largest<4>(v, count);
    if (lane == 0) s.bound = k;
  }
  __syncthreads();
  return s.bound;
}

// How many of the n things come before thing c, counted by `share` neighbouring lanes (a power of two up to
// 64), every one of which returns it.
template <class Before>
__device__ __forceinline__ uint32_t rank_of(int share, uint32_t n, Before before) {
  uint32_t rank = 0;
#pragma unroll 4
  for (uint32_t j = threadIdx.x & (share - 1); j < n; j += share) rank += before(j) ? 1u : 0u;
#pragma unroll
  for (int stride = 1; stride < 64; stride *= 2)
    if (stride < share) rank += xor_lane_by(rank, stride);
  return rank;
}
// The lanes to a thing where `lanes` of them rank n.
__device__ __forceinline__ int share_of(int lanes, uint32_t n) {
  int share = 1;
  while (share < 64 && n * share * 2 <= (uint32_t)lanes) share *= 2;
  return share;
}

// One workgroup of NW waves to a part of a row, every element read once. Many rows are bound by the issue of
// the 64-bit terms (16 operations an element) and by HBM, which one wave does not overlap: it asks for its next
// chunk before it looks at this one, but waits for it at the loop's end, and the unit's other waves cover that.
// 512 rows of 151,936 f32 in 65 us, 4.8 TB/s; the whole call 66, from f16 63, from bf16 59. Few rows are bound by
// latency: the load, the bound, the list, the ranks (four rows in 19 parts each: 7.7 us).
template <int DT, bool MASK, int NW>
__global__ __launch_bounds__(NW * 64) void beam_row_kernel(BeamArgs a) {
  using Reader = PartReader<DT, MASK>;
  constexpr int kBlockN = NW * 64;
  __shared__ BlockScratchT<NW> scratch;
  constexpr uint32_t kOwn = kListMax / NW;
  static_assert(kOwn >= kCountMax, "a full share holds as many as are kept");
  __shared__ __align__(8) uint32_t hist[kBins];
  __shared__ uint64_t list[kListMax];
  __shared__ uint32_t listed[NW];  // entries of each wave, those past its share too
  __shared__ BoundScratch<NW> bounds;
  __shared__ uint32_t held, bad, bound;
  __shared__ double wave_sum_[NW];
  __shared__ float wave_ref[NW], wave_max_[NW];
  uint64_t *const packed = reinterpret_cast<uint64_t *>(hist);
  static_assert(kBins * sizeof(uint32_t) >= kBlockN * sizeof(uint64_t), "the entries that are ranked");
  const int row = (int)blockIdx.x / a.parts, part = (int)blockIdx.x - row * a.parts;
  const int t = (int)threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int begin = part * a.part_len, len = min(a.part_len, a.vocab - begin);
  const Reader reader(a, row, begin, len);
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
  if (t < NW) listed[t] = 0;
  if (t == 0) {
    held = 0;
    bad = 0;
    bound = kNegInfKey + 1;
  }
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
  // The first bound, from the lanes' largest of the first chunks.
  uint32_t theta = max(bound_of<NW>(top == top ? key_of(top) : 0u, a.count, bounds), kNegInfKey + 1);

  double sum = 0.0;
  float ref = -INFINITY, largest = -INFINITY;  // terms are exp(x - ref)
  uint64_t *const own = list + wave * kOwn;
  uint32_t mine = 0;  // entries in it
  auto raise = [&](uint32_t k) {
    if (k > theta) {
      theta = k;
      if (lane == 0) atomicMax(&bound, k);
    }
  };
  auto take = [&]() {
    // Elements at or above the bound join the wave's list; a NaN is neither.
    if (__ballot(!(top < value_of(theta)))) {
      if (!(top < INFINITY)) bad = 1;
      // Where many lanes have one, the count-th largest of the lanes' maxima is a better bound.
      if (a.count <= 64 && __popcll(__ballot(top >= value_of(theta))) > a.count) {
        uint32_t v[1] = {top == top ? key_of(top) : 0u};
        raise(kth_largest<1>(v, a.count));
      }
      const float least = value_of(theta);
      const uint32_t before = mine;
#pragma unroll
      for (int i = 0; i < kLane; ++i) {
        const uint64_t who = __ballot(x[i] >= least);
        if (who) {
          const uint32_t to = mine + lanes_before(who);
          if (x[i] >= least && to < kOwn) own[to] = composite(key_of(x[i]), (uint32_t)reader.element(c, i));
          mine += (uint32_t)__popcll(who);
        }
      }
      // All lanes' entries before their count: a wave that sees the count reads them.
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
      if (lane == 0) __hip_atomic_store(&listed[wave], mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      // Now and then the count-th largest of all waves' last entries, 64 or 256, is a new bound.
      constexpr uint32_t kFew = 64 / NW, kMany = 256 / NW;
      const uint32_t span = a.count <= 32 ? kFew : kMany;
      if (before / span != mine / span && mine <= kOwn && c + NW < reader.chunks) {
        auto entry = [&](uint32_t i) {
          const uint32_t w = i / span, back = i % span + 1;
          const uint32_t n = min(__hip_atomic_load(&listed[w], __ATOMIC_ACQUIRE, __HIP_MEMORY_SCOPE_WORKGROUP), kOwn);
          return back <= n ? composite_key(list[w * kOwn + (n - back)]) : 0u;
        };
        if (span == kFew) {
          uint32_t v[1] = {entry(lane)};
          raise(kth_largest<1>(v, a.count));
        } else {
          uint32_t v[4] = {entry(lane), entry(64 + lane), entry(128 + lane), entry(192 + lane)};
          raise(kth_largest<4>(v, a.count));
        }
      }
    }
    if (__ballot(top - ref > 600.0f)) {
      // The first chunk with an element, or one far above: another reference. (The difference is rounded near 600
      // only; ref + 600 would be 1,024 above a ref of 2^33.)
      const float m = wave_max(top);
      if (m < INFINITY) {
        sum *= exp_or_none((double)ref - (double)m);
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
      for (int i = 0; i < kLane; ++i) part_sum[i & 1] += exp_or_none((double)x[i] - at);
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
    const uint32_t shared = __hip_atomic_load(&bound, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    reader.widen(raw, c, x);
    top = chunk_max();
    theta = max(theta, shared);
  }
  largest = wave_max(largest);
  sum = wave_sum(sum);
  if (lane == 0) {
    wave_sum_[wave] = sum;
    wave_ref[wave] = ref;
    wave_max_[wave] = largest;
  }
  __syncthreads();
  // The entries at or above the last bound, which at least `count` reach where there are so many.
  bool spilled = false;
  for (int w = 0; w < NW; ++w) spilled |= listed[w] > kOwn;
  const uint32_t last = max(bound, theta);
  for (uint32_t i = 0; i < min(mine, kOwn); i += 64) {
    const uint64_t v = i + lane < min(mine, kOwn) ? own[i + lane] : 0;
    const bool in = composite_key(v) >= last;
    const uint64_t who = __ballot(in);
    if (!who) continue;
    uint32_t at = 0;
    if (lane == 0) at = atomicAdd(&held, (uint32_t)__popcll(who));
    at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + lanes_before(who);
    if (in && at < (uint32_t)kBlockN) packed[at] = v;
  }
  __syncthreads();
  const uint32_t n = spilled ? ~0u : held;  // more than a wave's share: more than are kept
  if (bad || n == 0) {
    if (t == 0) a.sums[blockIdx.x] = RowSum{0.0, -INFINITY, 0, bad ? 1 : 0, 0};
    return;
  }
  const uint32_t need = min(n, (uint32_t)a.count);
  uint64_t *out = a.entries + (int64_t)blockIdx.x * a.count;
  if (wave == 0) {
    const float m = wave_max(lane < NW ? wave_max_[lane] : -INFINITY);
    double term = lane < NW ? wave_sum_[lane] : 0.0;
    if (term > 0.0) term *= exp_or_none((double)wave_ref[lane] - (double)m);
    term = wave_sum(term);
    if (t == 0) a.sums[blockIdx.x] = RowSum{term, m, (int)need, 0, 0};
  }
  if (n <= (uint32_t)kBlockN) {
    const int share = share_of(kBlockN, n);
    const uint32_t i = (uint32_t)t / share;
    const uint64_t v = i < n ? packed[i] : 0;
    const uint32_t rank = rank_of(share, n, [&](uint32_t j) { return packed[j] > v; });
    if (i < n && rank < need) out[rank] = v;
    return;
  }
  __syncthreads();
  auto pick = [&](auto for_each) {
    const SelectResult r = radix_select(for_each, need, hist, scratch);
    if (t == 0) scratch.slot = 0;
    __syncthreads();
    for_each([&](uint64_t v) {
      if (selected(v, r)) out[atomicAdd(&scratch.slot, 1u)] = v;
    });
  };
  if (!spilled) {
    pick([&](auto f) {
      for (uint32_t i = lane; i < mine; i += 64) f(own[i]);
    });
  } else {
    // A wave's share of the list does not hold what lies at or above its bounds: from the row again.
    const uint32_t *mask = a.allowed ? a.allowed + (int64_t)row * a.words : nullptr;
    const auto *src = reader.row;
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
  double sum = rs.count > 0 ? rs.sum * exp_or_none((double)rs.max - (double)m) : 0.0;
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
