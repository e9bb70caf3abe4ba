// Passes over rows of logits, shared by the operators that select from them: a reader of a part of a row, 64-bit
// exponentials, and the list of a part's first entries by (logit, index), kept while the part streams by.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "block_ops.h"
#include "device_math.h"
#include "elem.h"

namespace tabby {

constexpr int kVocabMax = 1 << 28;            // places in a row in 32 bits, with room
constexpr int kChunk = 1024;                  // elements a wave takes at a time
constexpr int kLane = kChunk / 64;            // of them to a lane

constexpr int kListCountMax = 128;            // entries that are kept
constexpr int kListMax = 4096;                // entries above the bound that LDS holds, a share to each wave

typedef uint32_t uint32x2 __attribute__((ext_vector_type(2)));

// a b + c, c a constant. HELD: written out, so that c stays in scalar registers, where the compiler copies it to vector ones first to
// add to it there: for kernels that have none to spare (the verification's decision spills 13 without it). The beam selection has, and
// takes 67 us with the copies and 70 without (64 groups of eight beams over 151,936 f32).
template <bool HELD>
__device__ __forceinline__ double fma_const(double a, double b, double c) {
  if constexpr (!HELD) return __builtin_fma(a, b, c);
  double r;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
  return r;
}

// 2^f in 64 bits for f in [-1/2, 1/2]: the polynomial of degree 7 through it at the Chebyshev nodes, within 5.5e-11 of it.
template <bool HELD = true>
__device__ __forceinline__ double exp2_64(double f) {
  double p = fma_const<HELD>(f, 1.530370102315244e-05, 0.0001546972921563772);
  p = fma_const<HELD>(p, f, 0.0013333478472326247);
  p = fma_const<HELD>(p, f, 0.009618025613309008);
  p = fma_const<HELD>(p, f, 0.055504109063275894);
  p = fma_const<HELD>(p, f, 0.24022651213498245);
  p = fma_const<HELD>(p, f, 0.6931471805568318);
  return fma_const<HELD>(p, f, 0.9999999999595618);
}

// exp(d) in 64 bits for d in [-690, 690]: t = d log2(e) is split into the nearest whole number, found by adding
// and taking away 1.5 * 2^52, whose low word then holds it, and the rest f in [-1/2, 1/2]. A sum of such terms
// decides the order of two beams' continuations only where their scores are that close.
template <bool HELD = true>
__device__ __forceinline__ double exp_64(double d) {
  constexpr double kLog2e = 1.4426950408889634;
  const double magic = 6755399441055744.0;
  const double shifted = __builtin_fma(d, kLog2e, magic);
  uint32x2 bits = __builtin_bit_cast(uint32x2, exp2_64<HELD>(__builtin_fma(d, kLog2e, -(shifted - magic))));
  bits.y += __builtin_bit_cast(uint32x2, shifted).x << 20;
  return __builtin_bit_cast(double, bits);
}
// The same for any d <= 690, -inf too: below -690 nothing is left that a sum of at least 1 would hold. Above 690 the
// exponent's field runs over, and the result, NaN included, has nothing to do with exp.
template <bool HELD = true>
__device__ __forceinline__ double exp_or_none(double d) { return exp_64<HELD>(fmax(d, -690.0)); }

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

  // mask_: the row's words, `words_` of them; null where there is none.
  __device__ __forceinline__ PartReader(const Bits *row_, const uint32_t *mask_, int words_, int begin_, int len_)
      : row(row_), mask(mask_), begin(begin_), len(len_), words(words_), chunks((len_ + kChunk - 1) / kChunk) {}

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

// The first `count` entries of a part by (logit, index), each element seen once. A bound, the count-th largest of 64
// (256) columns' maxima of the first chunks, lets through what can matter; each wave lists that for itself, and
// every few entries the waves' last ones give a better bound. A list that runs over has its part read again.
template <int NW>
struct ListScratch {
  BlockScratchT<NW> block;
  __attribute__((aligned(8))) uint32_t hist[kBins];
  uint64_t list[kListMax];
  uint32_t listed[NW];  // entries of each wave, those past its share too
  BoundScratch<NW> bounds;
  uint32_t held, bad, bound;
};

template <int NW>
struct RowList {
  static constexpr int kThreads = NW * 64;
  static constexpr uint32_t kOwn = kListMax / NW;
  static_assert(kOwn >= kListCountMax, "a full share holds as many as are kept");
  static_assert(kBins * sizeof(uint32_t) >= kThreads * sizeof(uint64_t), "the entries that are ranked");

  ListScratch<NW> &s;
  uint64_t *const own;
  const int count, wave, lane;
  uint32_t mine = 0;  // entries in `own`
  uint32_t theta;     // the bound that this wave goes by

  // By the whole workgroup; `top` is the largest of the lane's first elements, NaN if one of them is.
  __device__ __forceinline__ RowList(ListScratch<NW> &s_, int count_, int wave_, float top)
      : s(s_), own(s_.list + wave_ * kOwn), count(count_), wave(wave_), lane(wave_lane()) {
    const int t = (int)threadIdx.x;
    if (t < NW) s.listed[t] = 0;
    if (t == 0) {
      s.held = 0;
      s.bad = 0;
      s.bound = kNegInfKey + 1;
    }
    theta = max(bound_of<NW>(top == top ? key_of(top) : 0u, count, s.bounds), kNegInfKey + 1);
  }

  __device__ __forceinline__ void raise(uint32_t k) {
    if (k > theta) {
      theta = k;
      if (lane == 0) atomicMax(&s.bound, k);
    }
  }
  __device__ __forceinline__ uint32_t shared_bound() const {
    return __hip_atomic_load(&s.bound, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  }

  // Chunk c's elements x at or above the bound join the wave's list; a NaN is neither. `top` is their largest.
  template <class Reader>
  __device__ __forceinline__ void take(const Reader &reader, int c, const float (&x)[kLane], float top) {
    if (!__ballot(!(top < value_of(theta)))) return;
    if (!(top < INFINITY)) s.bad = 1;
    // Where many lanes have one, the count-th largest of the lanes' maxima is a better bound.
    if (count <= 64 && __popcll(__ballot(top >= value_of(theta))) > count) {
      uint32_t v[1] = {top == top ? key_of(top) : 0u};
      raise(kth_largest<1>(v, count));
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
    if (lane == 0) __hip_atomic_store(&s.listed[wave], mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    // Now and then the count-th largest of all waves' last entries, 64 or 256, is a new bound.
    constexpr uint32_t kFew = 64 / NW, kMany = 256 / NW;
    const uint32_t span = count <= 32 ? kFew : kMany;
    if (before / span != mine / span && mine <= kOwn && c + NW < reader.chunks) {
      auto entry = [&](uint32_t i) {
        const uint32_t w = i / span, back = i % span + 1;
        const uint32_t n = min(__hip_atomic_load(&s.listed[w], __ATOMIC_ACQUIRE, __HIP_MEMORY_SCOPE_WORKGROUP), kOwn);
        return back <= n ? composite_key(s.list[w * kOwn + (n - back)]) : 0u;
      };
      if (span == kFew) {
        uint32_t v[1] = {entry(lane)};
        raise(kth_largest<1>(v, count));
      } else {
        uint32_t v[4] = {entry(lane), entry(64 + lane), entry(128 + lane), entry(192 + lane)};
        raise(kth_largest<4>(v, count));
      }
    }
  }

  // After a barrier that follows every wave's last take: packs the entries at or above the last bound, which at
  // least `count` reach where there are so many, and returns their number; ~0 if a wave's share ran over.
  __device__ __forceinline__ uint32_t pack() {
    uint64_t *const packed = reinterpret_cast<uint64_t *>(s.hist);
    bool spilled = false;
    for (int w = 0; w < NW; ++w) spilled |= s.listed[w] > kOwn;
    const uint32_t last = max(s.bound, theta);
    for (uint32_t i = 0; i < min(mine, kOwn); i += 64) {
      const uint64_t v = i + lane < min(mine, kOwn) ? own[i + lane] : 0;
      const bool in = composite_key(v) >= last;
      const uint64_t who = __ballot(in);
      if (!who) continue;
      uint32_t at = 0;
      if (lane == 0) at = atomicAdd(&s.held, (uint32_t)__popcll(who));
      at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + lanes_before(who);
      if (in && at < (uint32_t)kThreads) packed[at] = v;
    }
    __syncthreads();
    return spilled ? ~0u : s.held;  // more than a wave's share: more than are kept
  }

  // The first `need` of pack()'s n entries to out; in order where n is at most kThreads. `each` visits all of the
  // part's entries above -inf, for a share that ran over.
  template <class Each>
  __device__ __forceinline__ void select(uint32_t n, uint32_t need, uint64_t *out, Each each) {
    const uint64_t *const packed = reinterpret_cast<const uint64_t *>(s.hist);
    const int t = (int)threadIdx.x;
    if (n <= (uint32_t)kThreads) {
      const int share = share_of(kThreads, n);
      const uint32_t i = (uint32_t)t / share;
      const uint64_t v = i < n ? packed[i] : 0;
      const uint32_t rank = rank_of(share, n, [&](uint32_t j) { return packed[j] > v; });
      if (i < n && rank < need) out[rank] = v;
      return;
    }
    __syncthreads();
    auto pick = [&](auto for_each) {
      const SelectResult r = radix_select(for_each, need, s.hist, s.block);
      if (t == 0) s.block.slot = 0;
      __syncthreads();
      for_each([&](uint64_t v) {
        if (selected(v, r)) out[atomicAdd(&s.block.slot, 1u)] = v;
      });
    };
    if (n != ~0u) {
      pick([&](auto f) {
        for (uint32_t i = lane; i < mine; i += 64) f(own[i]);
      });
    } else {
      pick(each);
    }
  }
};

// The largest of a lane's elements, NaN if one of them is.
__device__ __forceinline__ float chunk_max(const float (&x)[kLane]) {
  float m = x[0];
#pragma unroll
  for (int i = 1; i < kLane; ++i) m = max_or_nan(m, x[i]);
  return m;
}

}  // namespace tabby
