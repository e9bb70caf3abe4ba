// Verification of drafted tokens (speculative decoding): how many of a request's drafted tokens its target accepts,
// and the token that follows them.
//
// Request r has n drafted tokens d_1 .. d_n, n + 1 rows of the target's logits (row j: after j of the tokens) and, unless the
// tokens were certain, the n rows of logits that they were drawn from. P_j and Q_j are the distributions that the sampler
// draws from under the request's settings: the first top_k entries by (logit, lower index), weights exp((x - max) / T), cut
// after the first at which their running sum reaches top_p of the total, divided by what is left; T <= 0: the first entry.
// d_j+1 is accepted while
//   u_j Q_j(d_j+1) < P_j(d_j+1)          (Q = 1 where the tokens were certain)
// and the token after the last accepted one is drawn from max(P_j - Q_j, 0), divided by its sum, at the first refusal, from
// P_n if there is none: the first token in the vocabulary's order at which the running sum exceeds u of the total. What
// comes out is distributed as if every token had been drawn from the target.
//
// Kernels, in order:
//   rows    a workgroup to a part of a row: the list of its first entries (top_k up to 128), or its maximum and the sum of
//           exp((x - max) / T) (the whole vocabulary, or larger pools)
//   settle  a workgroup to a row: its parts together, the cut, and the probability of its drafted token. A distribution
//           is then a maximum, a total and a threshold: an entry is in it if its (logit, index) is at or above that
//   decide  a workgroup to a request: how many are accepted; pools are drawn from here
//   weigh   (whole vocabularies) a workgroup to a segment of a deciding row: the sum of what is drawn from
//   pick    (whole vocabularies) a workgroup to a request: the draw, among segments, then within one
// Sums are in 64 bits, and exponentials within 5.5e-11: which token comes out hangs on comparisons of sums.

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

constexpr int kPoolMax = kListCountMax;       // entries of a pool that is kept as a list
constexpr int kDraftsMax = 63;                // of a request: one wave decides
constexpr int kVerifyVocabMax = 1 << 24;      // masses of a row's entries are added up as whole multiples of 2^-38 or less
constexpr int64_t kBlocksMax = (1 << 22) - 1;  // of 1,024 threads each
constexpr int kPartsMax = 32;
constexpr int kSegment = 4096;                // elements of a segment

enum Kind : int32_t { kInvalid = 0, kGreedy, kPool, kWhole };

// What `rows` leaves of a part.
struct PartSum {
  double sum;     // of exp((x - max) / T)
  float max;
  int32_t count;  // entries written
  int32_t bad;    // a NaN or +inf
  int32_t reserved;
};

// A row's distribution.
struct RowDist {
  double total;        // of the weights exp((x - max) / T) that are left
  double drafted;      // the drafted token's probability; below 0: there is no such token
  uint64_t threshold;  // the last entry's composite
  float max;
  int32_t count;       // a pool's entries that are left
  int32_t bad;         // a NaN, +inf, or nothing above -inf
  int32_t reserved;
};

enum Draw : int32_t { kDone = 0, kFromTarget, kFromRest, kWithoutToken };

struct Decision {
  int32_t accepted;
  int32_t draw;
};

struct VerifyArgs {
  const void *logits, *draft_logits;  // draft_logits may be null
  int64_t stride, draft_stride;
  const int32_t *drafts;
  const double *uniforms;
  const int32_t *offsets;  // [requests + 1] or null
  const tabby_row_params *params;
  int rows, requests, drafts_max, vocab, slots;
  bool whole;  // requests may draw from the whole vocabulary
  int parts, part_len, segments;
  int32_t *tokens, *accepted, *status;
  PartSum *sums;         // [requests][slots][parts]
  uint64_t *entries;     // [requests][slots][parts][kPoolMax]
  RowDist *dists;        // [requests][slots]
  uint64_t *pools;       // [requests][slots][kPoolMax]
  Decision *decisions;   // [requests]
  double2 *segment_sums;  // [requests][segments]: of max(P - Q, 0) and of P
};

struct Setting {
  Kind kind;
  int k;
  double inverse, top_p;
};

__device__ __forceinline__ Setting setting_of(const VerifyArgs &a, int request) {
  const tabby_row_params p = a.params[request];
  Setting s{kInvalid, 1, 1.0, p.top_p};
  if (!(p.temperature < (double)INFINITY) || p.top_k < 0 || p.reserved != 0) return s;
  if (p.temperature <= 0.0) {
    s.kind = kGreedy;
    return s;
  }
  s.k = p.top_k == 0 ? a.vocab : min(p.top_k, a.vocab);
  // Below 1e-290 two logits that differ at all are further apart than an exponential reaches, as they are at it.
  s.inverse = 1.0 / fmax(p.temperature, 1e-290);
  s.kind = s.k <= kPoolMax ? kPool : a.whole ? kWhole : kInvalid;
  return s;
}

// Where a request's rows lie; drafts < 0: nowhere.
struct Place {
  int first, drafts;  // the target's first row, the number of drafted tokens
  int first_draft;    // the first drafted token
};

__device__ __forceinline__ Place place_of(const VerifyArgs &a, int request) {
  const int64_t first = a.offsets ? a.offsets[request] : (int64_t)request * (a.drafts_max + 1);
  const int64_t last = a.offsets ? a.offsets[request + 1] : first + a.drafts_max + 1;
  const int64_t drafts = last - first - 1, first_draft = first - request;
  if (first < 0 || last > a.rows || drafts < 0 || drafts > a.drafts_max || first_draft < 0 ||
      first_draft + drafts > a.rows - a.requests)
    return {0, -1, 0};
  return {(int)first, (int)drafts, (int)first_draft};
}

// Slots 0 .. drafts_max are the target's rows, those after them the draft's.
struct SlotRow {
  bool used;
  int drafted;  // the token that the row's probability is asked for, or -1
  const void *base;
};

template <int DT>
__device__ __forceinline__ SlotRow row_of(const VerifyArgs &a, const Place &p, Kind kind, int slot) {
  using Bits = typename Elem<DT>::Bits;
  const bool target = slot <= a.drafts_max;
  const int j = target ? slot : slot - (a.drafts_max + 1);
  if (kind == kInvalid || p.drafts < 0 || j > p.drafts || (!target && (j == p.drafts || kind == kGreedy))) return {false, -1, nullptr};
  const Bits *base = target ? (const Bits *)a.logits + (int64_t)(p.first + j) * a.stride
                            : (const Bits *)a.draft_logits + (int64_t)(p.first_draft + j) * a.draft_stride;
  return {true, j < p.drafts ? p.first_draft + j : -1, base};
}

template <int DT, int NW>
__global__ __launch_bounds__(NW * 64) void verify_rows_kernel(VerifyArgs a) {
  using Reader = PartReader<DT, false>;
  __shared__ ListScratch<NW> scratch;
  __shared__ double wave_sums[NW];
  __shared__ float wave_refs[NW], wave_tops[NW];
  const int row = (int)blockIdx.x / a.parts, part = (int)blockIdx.x - row * a.parts;
  const int request = row / a.slots, slot = row - request * a.slots;
  const int t = (int)threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const Setting set = setting_of(a, request);
  const SlotRow source = row_of<DT>(a, place_of(a, request), set.kind, slot);
  if (!source.used) return;
  const int begin = part * a.part_len, len = min(a.part_len, a.vocab - begin);
  PartSum *const out = a.sums + blockIdx.x;
  const Reader reader((const typename Reader::Bits *)source.base, nullptr, 0, begin, len);
  typename Reader::Raw raw, next;
  float x[kLane];
  int c = wave;
  reader.load(c, raw);
  reader.load(c + NW, next);
  float top = -INFINITY;  // of the lane's elements of the chunk; NaN if one of them is
  if (c < reader.chunks) {
    reader.widen(raw, c, x);
    top = chunk_max(x);
  } else {
#pragma unroll
    for (int i = 0; i < kLane; ++i) x[i] = -INFINITY;
  }
  // The next chunk's elements, until there are none.
  auto advance = [&]() {
    c += NW;
    raw = next;
    if (c >= reader.chunks) return false;
    reader.load(c + NW, next);
    reader.widen(raw, c, x);
    top = chunk_max(x);
    return true;
  };
  if (set.kind != kWhole) {
    RowList<NW> list(scratch, set.k, wave, top);
    float largest = -INFINITY;
    if (c < reader.chunks) {
      for (;;) {
        list.take(reader, c, x, top);
        largest = fmaxf(largest, top);
        const uint32_t shared = list.shared_bound();
        if (!advance()) break;
        list.theta = max(list.theta, shared);
      }
    }
    largest = wave_max(largest);
    if (lane == 0) wave_tops[wave] = largest;
    __syncthreads();
    const uint32_t n = list.pack();
    if (scratch.bad || n == 0) {
      if (t == 0) *out = PartSum{0.0, -INFINITY, 0, scratch.bad ? 1 : 0, 0};
      return;
    }
    const uint32_t need = min(n, (uint32_t)set.k);
    if (wave == 0) {
      const float m = wave_max(lane < NW ? wave_tops[lane] : -INFINITY);
      if (t == 0) *out = PartSum{0.0, m, (int)need, 0, 0};
    }
    list.select(n, need, a.entries + (int64_t)blockIdx.x * kPoolMax, [&](auto f) {
      for (int e = begin + t; e < begin + len; e += NW * 64) {
        const float v = Reader::E::widen(reader.row[e]);
        if (v > -INFINITY) f(composite(key_of(v), (uint32_t)e));
      }
    });
    return;
  }
  double sum = 0.0;
  float ref = -INFINITY, largest = -INFINITY;  // terms are exp((x - ref) / T)
  bool bad = false;
  if (c < reader.chunks) {
    do {
      bad |= !(top < INFINITY);
      if (__ballot(!(((double)top - (double)ref) * set.inverse <= 600.0))) {
        // The first chunk with an element, or one far above: another reference.
        const float m = wave_max(top);
        if (m > ref && m < INFINITY) {
          if (ref > -INFINITY) sum *= exp_or_none(((double)ref - (double)m) * set.inverse);
          ref = m;
        }
      }
      largest = fmaxf(largest, top);
      // A chunk whose terms are all below e^-50 adds nothing that the sum would hold.
      if (ref > -INFINITY && __ballot(((double)top - (double)ref) * set.inverse >= -50.0)) {
        const double at = (double)ref;
        double part_sum[2] = {0.0, 0.0};
#pragma unroll
        for (int i = 0; i < kLane; ++i) part_sum[i & 1] += exp_or_none(((double)x[i] - at) * set.inverse);
        sum += part_sum[0] + part_sum[1];
      }
    } while (advance());
  }
  bad = __ballot(bad) != 0;
  largest = wave_max(largest);
  sum = wave_sum(sum);
  if (lane == 0) {
    wave_sums[wave] = sum;
    wave_refs[wave] = ref;
    wave_tops[wave] = bad ? INFINITY : largest;
  }
  __syncthreads();
  if (wave == 0) {
    const float m = wave_max(lane < NW ? wave_tops[lane] : -INFINITY);
    double term = lane < NW ? wave_sums[lane] : 0.0;
    if (term > 0.0) term *= exp_or_none(((double)wave_refs[lane] - (double)m) * set.inverse);
    term = wave_sum(term);
    if (t == 0) *out = m < INFINITY ? PartSum{term, m, 0, 0, 0} : PartSum{0.0, -INFINITY, 0, 1, 0};
  }
}

// A pool's weights run off by 1e-15 from the sampler's own exponential; a whole vocabulary's as its sums do.
__device__ __forceinline__ double weight_of(float x, float max, double inverse) {
  return exp_nonpos(((double)x - (double)max) * inverse);
}

// Inclusive prefix sum over the wave's lanes, always in the same order.
template <typename T>
__device__ __forceinline__ T wave_prefix(T v) {
  const int lane = wave_lane();
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const T o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// The same over a workgroup's threads, in their order; `total` is that of all of them. `scratch` holds NW values and may
// be used again after the workgroup has met.
template <int NW, typename T>
__device__ __forceinline__ T block_prefix(T v, T *scratch, T &total) {
  const int wave = (int)threadIdx.x >> 6;
  v = wave_prefix(v);
  __syncthreads();
  if (wave_lane() == 63) scratch[wave] = v;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < wave) before += scratch[w];
    total += scratch[w];
  }
  return before + v;
}

constexpr int kSettleWaves = 16;
constexpr int kSettleThreads = kSettleWaves * 64;
constexpr int kHeldMax = kPartsMax * kPoolMax;  // entries that a settling workgroup holds
static_assert(kHeldMax == 4096, "a power of two: they are sorted");

// Masses of a row's entries are whole multiples of 2^-shift: their sums are exact and do not depend on an order.
__device__ __forceinline__ int mass_shift(int vocab) { return 62 - (32 - __clz(vocab)); }
__device__ __forceinline__ uint64_t mass_of(float x, float max, double inverse, double unit) {
  return (uint64_t)(exp_or_none(((double)x - (double)max) * inverse) * unit + 0.5);
}

// The bin of an entry `below` the row's maximum, in temperatures: 128 to a doubling of 1 + below, the largest
// entries in the highest. Equal logits share one, and a larger logit has none below a smaller one's.
__device__ __forceinline__ uint32_t bin_of(float x, float max, float inverse) {
  const float below = (max - x) * inverse + 1.0f;
  const uint32_t at = (__float_as_uint(below) - 0x3f800000u) >> 16;
  return (uint32_t)(kBins - 1) - min(at, (uint32_t)(kBins - 1));
}

struct SettleScratch {
  __attribute__((aligned(16))) uint64_t held[kHeldMax];
  uint64_t masses[kBins];
  uint32_t counts[kBins];
  BlockScratchT<kSettleWaves> block;
  BoundScratch<kSettleWaves> bounds;
  uint64_t wave64[kSettleWaves];
  uint64_t found_mass, found_entry;
  uint32_t found_bin, found_above, taken;
};

// Every element of a row above -inf, and its place.
template <int DT, class F>
__device__ __forceinline__ void each_element(const void *base, int vocab, F f) {
  using E = Elem<DT>;
  const typename E::Bits *row = (const typename E::Bits *)base;
  constexpr int kAhead = 4;
  const int whole = vocab / E::kVec;
  for (int i = (int)threadIdx.x; i < whole; i += kAhead * kSettleThreads) {
    u32x4 raw[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      raw[u] = *reinterpret_cast<const u32x4_any *>(row + (int64_t)min(i + u * kSettleThreads, whole - 1) * E::kVec);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i + u * kSettleThreads >= whole) break;
      float v[E::kVec];
      E::widen16(raw[u], v);
#pragma unroll
      for (int j = 0; j < E::kVec; ++j)
        if (v[j] > -INFINITY) f(v[j], (uint32_t)((i + u * kSettleThreads) * E::kVec + j));
    }
  }
  for (int e = whole * E::kVec + (int)threadIdx.x; e < vocab; e += kSettleThreads) {
    const float v = E::widen(row[e]);
    if (v > -INFINITY) f(v, (uint32_t)e);
  }
}

// The highest bin at which the running count, or mass, from the highest on reaches `need`: its place, and what lies above
// it. (A need that no bin reaches: the lowest one that holds anything.)
template <typename T>
__device__ __forceinline__ void find_reached(const T *bins, T need, T *wave_space, SettleScratch &s, T *above) {
  constexpr int kPer = kBins / kSettleThreads;
  const int t = (int)threadIdx.x, high = kBins - 1 - t * kPer;
  T own[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    own[i] = bins[high - i];
    sum += own[i];
  }
  T total;
  T before = block_prefix<kSettleWaves>(sum, wave_space, total) - sum;
  const T goal = need < total ? need : total;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    // The first at which the sum reaches the goal: bins that hold nothing do not change it.
    if (own[i] > 0 && before < goal && before + own[i] >= goal) {
      s.found_bin = (uint32_t)(high - i);
      *above = before;
    }
    before += own[i];
  }
  __syncthreads();
}

// The entries of one bin, or of a part of one: those whose composite begins with `prefix` down to bit `done`.
struct Cell {
  uint32_t bin;
  int done;  // 64: all of the bin
  uint64_t prefix;
  __device__ __forceinline__ bool holds(uint64_t c) const { return done == 64 || (c >> done) == (prefix >> done); }
};

// What a row's cut has come to: entries down to and with `entry`, and their mass.
struct Cut {
  uint64_t entry;
  uint64_t mass;
};

// The row cut after its k-th entry (BY_MASS: after the first at which the running mass reaches `goal`), given the bins'
// counts and masses, and no further than `last`.
template <int DT, bool BY_MASS>
__device__ __forceinline__ Cut cut_row(const VerifyArgs &a, const void *base, const Setting &set, float max, uint32_t k, uint64_t goal,
                                       uint64_t last, SettleScratch &s) {
  const int t = (int)threadIdx.x;
  const float inverse = fminf((float)set.inverse, 3.0e38f);
  const double unit = __builtin_ldexp(1.0, mass_shift(a.vocab));
  uint64_t above_mass = 0;  // of what lies above the cell
  uint32_t above = 0;
  Cell cell{0, 64, 0};
  uint32_t in_cell;
  auto descend = [&]() {
    // Where the goal is reached among the bins of s, and what lies above it.
    if constexpr (BY_MASS) {
      const uint64_t left = goal > above_mass ? goal - above_mass : 1;
      find_reached<uint64_t>(s.masses, left, s.wave64, s, &s.found_mass);
      above_mass += s.found_mass;
    } else {
      find_reached<uint32_t>(s.counts, k - above, s.block.u, s, &s.found_above);
      above += s.found_above;
      // Their mass: of the bins above.
      uint64_t mass = 0, total;
      for (int b = kBins - 1 - t; b > (int)s.found_bin; b -= kSettleThreads) mass += s.masses[b];
      block_prefix<kSettleWaves>(mass, s.wave64, total);
      above_mass += total;
    }
    in_cell = s.counts[s.found_bin];
    const uint32_t found = s.found_bin;
    __syncthreads();
    return found;
  };
  cell.bin = descend();
  // More entries than LDS holds: the next eleven bits of their composites.
  while (in_cell > (uint32_t)kHeldMax && cell.done > 0) {
    const int shift = cell.done >= 11 ? cell.done - 11 : 0;
    const uint32_t digits = (1u << (cell.done - shift)) - 1;
    for (int b = t; b < kBins; b += kSettleThreads) {
      s.counts[b] = 0;
      s.masses[b] = 0;
    }
    __syncthreads();
    each_element<DT>(base, a.vocab, [&](float x, uint32_t e) {
      if (bin_of(x, max, inverse) != cell.bin) return;
      const uint64_t c = composite(key_of(x), e);
      if (c < last || !cell.holds(c)) return;
      const uint32_t digit = (uint32_t)(c >> shift) & digits;
      atomicAdd(&s.counts[digit], 1u);
      atomicAdd((unsigned long long *)&s.masses[digit], (unsigned long long)mass_of(x, max, set.inverse, unit));
    });
    __syncthreads();
    const uint32_t digit = descend();
    cell.prefix |= (uint64_t)digit << shift;
    cell.done = shift;
  }
  if (t == 0) s.taken = 0;
  __syncthreads();
  each_element<DT>(base, a.vocab, [&](float x, uint32_t e) {
    if (bin_of(x, max, inverse) != cell.bin) return;
    const uint64_t c = composite(key_of(x), e);
    if (c < last || !cell.holds(c)) return;
    const uint32_t at = atomicAdd(&s.taken, 1u);
    if (at < (uint32_t)kHeldMax) s.held[at] = c;
  });
  __syncthreads();
  const int n = (int)min(s.taken, (uint32_t)kHeldMax), room = next_pow2(n);
  for (int i = n + t; i < room; i += kSettleThreads) s.held[i] = 0;
  __syncthreads();
  bitonic_sort_desc<kSettleWaves>(s.held, room);
  if (room <= 1) __syncthreads();
  // In order, four to a thread: the first that reaches the goal, or the last there is.
  constexpr int kPer = kHeldMax / kSettleThreads;
  uint64_t mass[kPer], sum = 0, total;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = t * kPer + i;
    mass[i] = at < n ? mass_of(value_of(composite_key(s.held[at])), max, set.inverse, unit) : 0;
    sum += mass[i];
  }
  uint64_t before = block_prefix<kSettleWaves>(sum, s.wave64, total) - sum + above_mass;
  const uint64_t reach = BY_MASS ? (goal < above_mass + total ? goal : above_mass + total) : 0;
  bool reached = BY_MASS && t > 0 && before >= reach;  // by an entry of a thread before this one
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = t * kPer + i;
    before += mass[i];
    const bool here = at < n && (BY_MASS ? !reached && before >= reach : above + at + 1 == k || (at == n - 1 && above + n < k));
    if (here) {
      s.found_entry = s.held[at];
      s.found_mass = before;
      reached = true;
    }
  }
  __syncthreads();
  return {s.found_entry, s.found_mass};
}

template <int DT>
__global__ __launch_bounds__(kSettleThreads) void verify_settle_kernel(VerifyArgs a) {
  using E = Elem<DT>;
  __shared__ SettleScratch s;
  const int row = (int)blockIdx.x;
  const int request = row / a.slots, slot = row - request * a.slots;
  const int t = (int)threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const Setting set = setting_of(a, request);
  const SlotRow source = row_of<DT>(a, place_of(a, request), set.kind, slot);
  if (!source.used) return;
  const PartSum *sums = a.sums + (int64_t)row * a.parts;
  RowDist dist{0.0, 0.0, 0, -INFINITY, 0, 0, 0};
  float m = -INFINITY;
  int bad = 0;
  for (int p = 0; p < a.parts; ++p) {
    m = fmaxf(m, sums[p].max);
    bad |= sums[p].bad;
  }
  bad |= !(m > -INFINITY);
  dist.max = m;
  dist.bad = bad;
  if (bad) {
    if (t == 0) a.dists[row] = dist;
    return;
  }
  if (set.kind == kWhole) {
    double total = 0.0;
    for (int p = 0; p < a.parts; ++p)
      if (sums[p].max > -INFINITY) total += sums[p].sum * exp_or_none(((double)sums[p].max - (double)m) * set.inverse);
    dist.total = total;
    const bool cut = set.top_p < 1.0;
    if (cut || set.k < a.vocab) {
      const float inverse = fminf((float)set.inverse, 3.0e38f);
      const double unit = __builtin_ldexp(1.0, mass_shift(a.vocab));
      for (int b = t; b < kBins; b += kSettleThreads) {
        s.counts[b] = 0;
        s.masses[b] = 0;
      }
      __syncthreads();
      each_element<DT>(source.base, a.vocab, [&](float x, uint32_t) {
        const uint32_t b = bin_of(x, m, inverse);
        atomicAdd(&s.counts[b], 1u);
        atomicAdd((unsigned long long *)&s.masses[b], (unsigned long long)mass_of(x, m, set.inverse, unit));
      });
      __syncthreads();
      uint64_t mass = 0, all;
      for (int b = t; b < kBins; b += kSettleThreads) mass += s.masses[b];
      block_prefix<kSettleWaves>(mass, s.wave64, all);
      Cut c{0, all};
      if (set.k < a.vocab) {
        c = cut_row<DT, false>(a, source.base, set, m, (uint32_t)set.k, 0, 0, s);
        if (cut) {
          // The bins again, of what is left.
          __syncthreads();
          for (int b = t; b < kBins; b += kSettleThreads) {
            s.counts[b] = 0;
            s.masses[b] = 0;
          }
          __syncthreads();
          each_element<DT>(source.base, a.vocab, [&](float x, uint32_t e) {
            if (composite(key_of(x), e) < c.entry) return;
            const uint32_t b = bin_of(x, m, inverse);
            atomicAdd(&s.counts[b], 1u);
            atomicAdd((unsigned long long *)&s.masses[b], (unsigned long long)mass_of(x, m, set.inverse, unit));
          });
          __syncthreads();
        }
      }
      if (cut) {
        // The smallest whole number of units that is top_p of the total, within the rounding of that product (so that
        // 900 of 1,000 equal entries are 0.9 of them); at least one.
        const double share = fmax(ceil(set.top_p * (double)c.mass * (1.0 - 0x1p-51)), 1.0);
        c = cut_row<DT, true>(a, source.base, set, m, 0, (uint64_t)share, c.entry, s);
      }
      dist.threshold = c.entry;
      dist.total = (double)c.mass / unit;
    }
  } else {
    // The parts' entries: those at or above a bound are ranked by counting.
    const uint64_t *entries = a.entries + (int64_t)row * a.parts * kPoolMax;
    const int slots = a.parts * kPoolMax;
    constexpr int kEach = kHeldMax / kSettleThreads;
    uint64_t entry[kEach], best = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int at = i * kSettleThreads + t;
      entry[i] = at < slots && at % kPoolMax < sums[at / kPoolMax].count ? entries[at] : 0;
      best = max(best, entry[i]);
    }
    if (t == 0) s.taken = 0;
    uint32_t theta = 0;
    if (a.parts > 1) theta = bound_of<kSettleWaves>((uint32_t)(best >> 32), set.k, s.bounds);
    else __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const bool in = entry[i] != 0 && composite_key(entry[i]) >= theta;
      const uint64_t who = __ballot(in);
      if (!who) continue;
      uint32_t at = 0;
      if (lane == 0) at = atomicAdd(&s.taken, (uint32_t)__popcll(who));
      at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + lanes_before(who);
      if (in) s.held[at] = entry[i];
    }
    __syncthreads();
    const uint32_t n = s.taken, need = min(n, (uint32_t)set.k);
    uint64_t *const pool = s.masses;  // in order
    const int share = share_of(kSettleThreads, n);
    for (uint32_t i = (uint32_t)t / share; i < (n + kSettleThreads - 1) / kSettleThreads * kSettleThreads / share; i += kSettleThreads / share) {
      const uint64_t v = i < n ? s.held[i] : 0;
      const uint32_t rank = rank_of(share, n, [&](uint32_t j) { return s.held[j] > v; });
      if (i < n && rank < need && (t & (share - 1)) == 0) pool[rank] = v;
    }
    __syncthreads();
    if (wave == 0) {
      double w[2], sum[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t i = (uint32_t)(lane + 64 * h);
        w[h] = i >= need ? 0.0 : set.kind == kGreedy ? 1.0 : weight_of(value_of(composite_key(pool[i])), m, set.inverse);
        sum[h] = wave_prefix(w[h]);
      }
      sum[1] += __shfl(sum[0], 63);
      const double total = __shfl(sum[1], 63);
      uint32_t left = need;
      if (set.top_p < 1.0) {
        const uint64_t low = __ballot(sum[0] >= set.top_p * total), high = __ballot(sum[1] >= set.top_p * total);
        const uint32_t first = low ? (uint32_t)__builtin_ctzll(low) : high ? 64u + (uint32_t)__builtin_ctzll(high) : need - 1;
        left = min(first + 1, need);
      }
      const int at = (int)left - 1;
      const double low = __shfl(sum[0], at & 63), high = __shfl(sum[1], at & 63);
      dist.total = at < 64 ? low : high;
      dist.threshold = pool[at];
      dist.count = (int)left;
      uint64_t *out = a.pools + (int64_t)row * kPoolMax;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t i = (uint32_t)(lane + 64 * h);
        if (i < left) out[i] = pool[i];
      }
    }
  }
  if (t != 0) return;
  if (source.drafted >= 0) {
    const int token = a.drafts[source.drafted];
    if (token < 0 || token >= a.vocab) {
      dist.drafted = -1.0;
    } else {
      const float x = E::widen(((const typename E::Bits *)source.base)[token]);
      if (x > -INFINITY && composite(key_of(x), (uint32_t)token) >= dist.threshold)
        dist.drafted = (set.kind == kGreedy ? 1.0 : weight_of(x, m, set.inverse)) / dist.total;
    }
  }
  a.dists[row] = dist;
}

// One workgroup of two waves to a request.
constexpr int kDecideThreads = 128;

__global__ __launch_bounds__(kDecideThreads) void verify_decide_kernel(VerifyArgs a) {
  __shared__ uint64_t target[kPoolMax], draft[kPoolMax];
  __shared__ double rest[kPoolMax], all[kPoolMax], wave_space[2];
  __shared__ int accepted_, status_;
  __shared__ uint32_t ids[kPoolMax];
  __shared__ uint64_t overs[2], somes[2];
  const int request = (int)blockIdx.x, t = (int)threadIdx.x;
  const Setting set = setting_of(a, request);
  const Place place = place_of(a, request);
  const RowDist *dists = a.dists + (int64_t)request * a.slots;
  const bool drawn = a.draft_logits != nullptr && set.kind != kGreedy;  // else the drafted tokens were certain
  if (t < 64) {
    const bool asked = place.drafts >= 0 && t < place.drafts && set.kind != kInvalid;
    bool good = false, broken = false, unknown = false;
    if (asked) {
      const RowDist &p = dists[t];
      const double claim = drawn ? dists[a.drafts_max + 1 + t].drafted : 1.0;
      broken = p.bad || (drawn && dists[a.drafts_max + 1 + t].bad);
      unknown = !broken && p.drafted < 0.0;
      good = !broken && !unknown && a.uniforms[place.first_draft + t] * claim < p.drafted;
    }
    // Of the greedy settings the draft's distribution is not asked: a token is accepted if it is the largest's.
    const uint64_t goods = __ballot(good), brokens = __ballot(broken), unknowns = __ballot(unknown);
    if (t == 0) {
      int n = 0, status = TABBY_EINVAL;
      if (place.drafts >= 0 && set.kind != kInvalid) {
        n = min((int)__builtin_ctzll(~goods), place.drafts);  // lane 63 never has a token
        const uint64_t here = 1ull << n;
        status = (brokens & here) || (n == place.drafts && dists[n].bad) ? TABBY_EDOMAIN : (unknowns & here) ? TABBY_EINVAL : TABBY_OK;
      }
      accepted_ = n;
      status_ = status;
    }
  }
  __syncthreads();
  const int n = accepted_, status = status_;
  int32_t *tokens = a.tokens + (int64_t)request * (a.drafts_max + 1);
  if (t <= a.drafts_max && (status != TABBY_OK || t != n)) tokens[t] = status == TABBY_OK && t < n ? a.drafts[place.first_draft + t] : -1;
  if (t == 0) {
    a.accepted[request] = status == TABBY_OK ? n : 0;
    if (a.status) a.status[request] = status;
  }
  const bool refused = n < place.drafts;
  const Draw draw = !refused || set.kind == kGreedy ? kFromTarget : drawn ? kFromRest : kWithoutToken;
  if (t == 0 && a.whole) a.decisions[request] = {n, status == TABBY_OK && set.kind == kWhole ? draw : kDone};
  if (status != TABBY_OK || set.kind == kWhole) return;
  // A pool: what is left of the target's entries, in the vocabulary's order.
  const RowDist p = dists[n];
  if (set.kind == kGreedy) {
    if (t == 0) tokens[n] = (int32_t)composite_index(p.threshold);
    return;
  }
  const RowDist q = draw == kFromRest ? dists[a.drafts_max + 1 + n] : p;
  const uint64_t own = t < p.count ? a.pools[((int64_t)request * a.slots + n) * kPoolMax + t] : 0;
  target[t] = own;
  if (draw == kFromRest) draft[t] = t < q.count ? a.pools[((int64_t)request * a.slots + a.drafts_max + 1 + n) * kPoolMax + t] : 0;
  __syncthreads();
  const uint32_t id = composite_index(own);
  double share = 0.0, left = 0.0;
  uint32_t before = 0;
  if (t < p.count) {
    share = weight_of(value_of(composite_key(own)), p.max, set.inverse) / p.total;
    left = share;
    if (draw == kFromRest) {
      for (int j = 0; j < q.count; ++j)
        if (composite_index(draft[j]) == id) left = fmax(share - weight_of(value_of(composite_key(draft[j])), q.max, set.inverse) / q.total, 0.0);
    } else if (draw == kWithoutToken && (int)id == a.drafts[place.first_draft + n]) {
      left = 0.0;
    }
    for (int j = 0; j < p.count; ++j) before += composite_index(target[j]) < id ? 1u : 0u;
    rest[before] = left;
    all[before] = share;
    ids[before] = id;
  }
  __syncthreads();
  double total;
  double v = t < p.count ? rest[t] : 0.0;
  double sum = block_prefix<2>(v, wave_space, total);
  if (!(total > 0.0)) {  // nothing left: P is Q, but for roundings
    v = t < p.count ? all[t] : 0.0;
    sum = block_prefix<2>(v, wave_space, total);
  }
  // The first whose running sum exceeds the share; the last with a weight where none does.
  const double goal = a.params[request].uniform * total;
  const uint64_t over = __ballot(v > 0.0 && sum > goal), some = __ballot(v > 0.0);
  if ((t & 63) == 0) {
    overs[t >> 6] = over;
    somes[t >> 6] = some;
  }
  __syncthreads();
  if (t == 0) {
    int at = 0;
    if (overs[0]) at = __builtin_ctzll(overs[0]);
    else if (overs[1]) at = 64 + __builtin_ctzll(overs[1]);
    else if (somes[1]) at = 127 - __builtin_clzll(somes[1]);
    else if (somes[0]) at = 63 - __builtin_clzll(somes[0]);
    tokens[n] = (int32_t)ids[at];
  }
}

// What a request draws from, over the whole vocabulary.
template <int DT>
struct RestOf {
  using E = Elem<DT>;
  using Bits = typename E::Bits;
  const Bits *target, *draft;
  RowDist p, q;
  double inverse, of_p, of_q;
  Draw draw;
  int token;
  __device__ __forceinline__ RestOf(const VerifyArgs &a, int request, const Decision &d) {
    const Setting set = setting_of(a, request);
    const Place place = place_of(a, request);
    const RowDist *dists = a.dists + (int64_t)request * a.slots;
    draw = (Draw)d.draw;
    inverse = set.inverse;
    p = dists[d.accepted];
    target = (const Bits *)a.logits + (int64_t)(place.first + d.accepted) * a.stride;
    of_p = 1.0 / p.total;
    q = p;
    draft = target;
    of_q = 0.0;
    token = -1;
    if (draw == kFromRest) {
      q = dists[a.drafts_max + 1 + d.accepted];
      draft = (const Bits *)a.draft_logits + (int64_t)(place.first_draft + d.accepted) * a.draft_stride;
      of_q = 1.0 / q.total;
    } else if (draw == kWithoutToken) {
      token = a.drafts[place.first_draft + d.accepted];
    }
  }
  static __device__ __forceinline__ double share(const RowDist &d, double inverse, double scale, float x, int e) {
    if (!(x > -INFINITY) || composite(key_of(x), (uint32_t)e) < d.threshold) return 0.0;
    return exp_or_none(((double)x - (double)d.max) * inverse) * scale;
  }
  // The sums over this thread's 16 elements of a segment; each(element, rest, share).
  template <class F>
  __device__ __forceinline__ void each(int first, int vocab, F f) const {
    constexpr int kOwn = kSegment / 256;
    const int at = first + (int)threadIdx.x * kOwn;
#pragma unroll
    for (int g = 0; g < kOwn / E::kVec; ++g) {
      const int e = at + g * E::kVec;
      if (e >= vocab) break;
      float x[E::kVec], y[E::kVec];
      E::widen16(load_values<DT, false>(target, e, vocab), x);
      if (draw == kFromRest) E::widen16(load_values<DT, false>(draft, e, vocab), y);
#pragma unroll
      for (int j = 0; j < E::kVec; ++j) {
        if (e + j >= vocab) break;
        const double v = share(p, inverse, of_p, x[j], e + j);
        double left = v;
        if (draw == kFromRest) left = fmax(v - share(q, inverse, of_q, y[j], e + j), 0.0);
        else if (e + j == token) left = 0.0;
        f(e + j, left, v);
      }
    }
  }
};

template <int DT>
__global__ __launch_bounds__(256) void verify_weigh_kernel(VerifyArgs a) {
  __shared__ double wave_space[2][4];
  const int request = (int)blockIdx.y, segment = (int)blockIdx.x, t = (int)threadIdx.x;
  const Decision d = a.decisions[request];
  if (d.draw == kDone) return;
  const RestOf<DT> rest(a, request, d);
  double left = 0.0, all = 0.0;
  rest.each(segment * kSegment, a.vocab, [&](int, double r, double v) {
    left += r;
    all += v;
  });
  left = wave_sum(left);
  all = wave_sum(all);
  if ((t & 63) == 0) {
    wave_space[0][t >> 6] = left;
    wave_space[1][t >> 6] = all;
  }
  __syncthreads();
  if (t == 0) {
    double2 sums{0.0, 0.0};
    for (int w = 0; w < 4; ++w) {
      sums.x += wave_space[0][w];
      sums.y += wave_space[1][w];
    }
    a.segment_sums[(int64_t)request * a.segments + segment] = sums;
  }
}

template <int DT>
__global__ __launch_bounds__(256) void verify_pick_kernel(VerifyArgs a) {
  __shared__ double wave_space[4], before_;
  __shared__ int segment_, last_, token_;
  const int request = (int)blockIdx.x, t = (int)threadIdx.x;
  const Decision d = a.decisions[request];
  if (d.draw == kDone) return;
  const RestOf<DT> rest(a, request, d);
  const double2 *sums = a.segment_sums + (int64_t)request * a.segments;
  // A run of segments to a thread.
  const int per = (a.segments + 255) / 256, begin = min(t * per, a.segments), end = min(begin + per, a.segments);
  double own = 0.0, own_all = 0.0, total, total_all;
  for (int i = begin; i < end; ++i) {
    own += sums[i].x;
    own_all += sums[i].y;
  }
  double before = block_prefix<4>(own, wave_space, total) - own;
  const double before_all = block_prefix<4>(own_all, wave_space, total_all) - own_all;
  const bool plain = !(total > 0.0);  // nothing left: P is Q, but for roundings
  if (plain) {
    total = total_all;
    before = before_all;
  }
  const double goal = a.params[request].uniform * total;
  if (t == 0) {
    segment_ = a.segments;
    last_ = -1;
    token_ = a.vocab;
  }
  __syncthreads();
  // The first segment whose running sum exceeds the share; the last with a weight where none does.
  double at = before;
  int found = a.segments, last = -1;
  double found_before = 0.0, last_before = 0.0;
  for (int i = begin; i < end; ++i) {
    const double v = plain ? sums[i].y : sums[i].x;
    if (v > 0.0) {
      last = i;
      last_before = at;
      if (found == a.segments && at + v > goal) {
        found = i;
        found_before = at;
      }
    }
    at += v;
  }
  if (found < a.segments) atomicMin(&segment_, found);
  if (last >= 0) atomicMax(&last_, last);
  __syncthreads();
  const int chosen = segment_ < a.segments ? segment_ : max(last_, 0);
  if (found == chosen && segment_ < a.segments) before_ = found_before;
  else if (last == chosen && segment_ == a.segments) before_ = last_before;
  __syncthreads();
  const double base = before_;
  if (t == 0) last_ = -1;
  __syncthreads();
  double sum = 0.0, all;
  rest.each(chosen * kSegment, a.vocab, [&](int, double r, double v) { sum += plain ? v : r; });
  double run = block_prefix<4>(sum, wave_space, all) - sum + base;
  int first = a.vocab, some = -1;
  rest.each(chosen * kSegment, a.vocab, [&](int e, double r, double v) {
    const double w = plain ? v : r;
    run += w;
    if (w > 0.0) {
      some = e;
      if (first == a.vocab && run > goal) first = e;
    }
  });
  if (first < a.vocab) atomicMin(&token_, first);
  if (some >= 0) atomicMax(&last_, some);
  __syncthreads();
  if (t == 0) a.tokens[(int64_t)request * (a.drafts_max + 1) + d.accepted] = token_ < a.vocab ? token_ : max(last_, 0);
}

int check_verify_shape(int32_t requests, int32_t drafts_max, int32_t vocab) {
  if (requests < 1 || vocab < 1) return record_failure(TABBY_EINVAL, "requests and vocab must be >= 1");
  if (drafts_max < 0 || drafts_max > kDraftsMax)
    return record_failure(TABBY_EINVAL, "drafts_max must be between 0 and " + std::to_string(kDraftsMax) + ", got " + std::to_string(drafts_max));
  if (vocab > kVerifyVocabMax) return record_failure(TABBY_EINVAL, "vocab must be at most " + std::to_string(kVerifyVocabMax));
  if ((int64_t)requests * (2 * drafts_max + 1) > kBlocksMax || requests > 65535)
    return record_failure(TABBY_EINVAL, "requests must be at most 65535, and their rows at most " + std::to_string(kBlocksMax));
  return TABBY_OK;
}

constexpr int kCus = 256;       // an MI355X's compute units
constexpr int kPartMin = 8192;  // a chunk to each of eight waves

// Few rows are cut into parts, a workgroup each, until there is about one to a compute unit.
int verify_parts(int64_t rows, int vocab) {
  const int64_t parts = std::min<int64_t>({kCus / std::max<int64_t>(rows, 1), (vocab + kPartMin - 1) / kPartMin, kPartsMax});
  return (int)std::max<int64_t>(parts, 1);
}

int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// The workspace's arrays: where each begins, and the end.
struct Space { int64_t sums, entries, dists, pools, decisions, segments, end; };
Space space_of(int64_t requests, int64_t slots, int64_t lists, int64_t segments) {
  Space s;
  s.sums = 0;
  s.entries = s.sums + aligned(lists * (int64_t)sizeof(PartSum));
  s.dists = s.entries + aligned(lists * kPoolMax * 8);
  s.pools = s.dists + aligned(requests * slots * (int64_t)sizeof(RowDist));
  s.decisions = s.pools + aligned(requests * slots * kPoolMax * 8);
  s.segments = s.decisions + aligned(requests * (int64_t)sizeof(Decision));
  s.end = s.segments + aligned(requests * segments * (int64_t)sizeof(double2));
  return s;
}

template <int DT>
int launch_verify(const VerifyArgs &a, hipStream_t s) {
  const unsigned rows = (unsigned)(a.requests * a.slots), blocks = rows * (unsigned)a.parts;
  // Four or eight waves where they have a chunk each. Else, up to a workgroup for each compute unit, sixteen.
  if (a.part_len <= 4 * kChunk) hipLaunchKernelGGL((verify_rows_kernel<DT, 4>), dim3(blocks), dim3(256), 0, s, a);
  else if (blocks <= (unsigned)kCus && a.part_len > 8 * kChunk) hipLaunchKernelGGL((verify_rows_kernel<DT, 16>), dim3(blocks), dim3(1024), 0, s, a);
  else hipLaunchKernelGGL((verify_rows_kernel<DT, 8>), dim3(blocks), dim3(512), 0, s, a);
  TABBY_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL(verify_settle_kernel<DT>, dim3(rows), dim3(kSettleThreads), 0, s, a);
  TABBY_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL(verify_decide_kernel, dim3((unsigned)a.requests), dim3(kDecideThreads), 0, s, a);
  TABBY_HIP_CHECK(hipGetLastError());
  if (!a.whole) return TABBY_OK;
  hipLaunchKernelGGL(verify_weigh_kernel<DT>, dim3((unsigned)a.segments, (unsigned)a.requests), dim3(256), 0, s, a);
  TABBY_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL(verify_pick_kernel<DT>, dim3((unsigned)a.requests), dim3(256), 0, s, a);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

}  // namespace
}  // namespace tabby

using namespace tabby;

extern "C" int tabby_draft_workspace(int32_t requests, int32_t drafts_max, int32_t vocab, int64_t *bytes) {
  if (!bytes) return record_failure(TABBY_EINVAL, "null pointer");
  const int rc = check_verify_shape(requests, drafts_max, vocab);
  if (rc) return rc;
  // For these sizes and every smaller one: rows that are cut make at most kCus parts.
  const int64_t slots = 2 * drafts_max + 1, lists = std::max<int64_t>(requests * slots, kCus);
  *bytes = space_of(requests, slots, lists, ((int64_t)vocab + kSegment - 1) / kSegment).end;
  return TABBY_OK;
}

extern "C" int tabby_draft_verify_device(const void *logits_dev, int32_t dtype, int64_t row_stride, int32_t rows,
                                         const void *draft_logits_dev, int64_t draft_row_stride, const int32_t *drafts_dev,
                                         const double *uniforms_dev, const int32_t *offsets_dev, int32_t requests,
                                         int32_t drafts_max, int32_t vocab, const tabby_row_params *params_dev,
                                         int32_t *tokens_dev, int32_t *accepted_dev, int32_t *status_dev,
                                         void *workspace_dev, int64_t workspace_bytes, uint32_t flags, void *stream) {
  int rc = check_verify_shape(requests, drafts_max, vocab);
  if (rc) return rc;
  if (rows < requests || rows > (int64_t)requests * (drafts_max + 1))
    return record_failure(TABBY_EINVAL, "rows must be between requests and requests x (drafts_max + 1)");
  if (!offsets_dev && rows != (int64_t)requests * (drafts_max + 1))
    return record_failure(TABBY_EINVAL, "without offsets there are drafts_max + 1 rows to a request");
  const int64_t total = rows - requests;  // drafted tokens
  if (!logits_dev || !params_dev || !tokens_dev || !accepted_dev || !workspace_dev || (total && (!drafts_dev || !uniforms_dev)))
    return record_failure(TABBY_EINVAL, "null pointer");
  if (!known_dtype(dtype)) return record_failure(TABBY_EINVAL, "dtype must be TABBY_F32, TABBY_F16 or TABBY_BF16");
  if ((rows > 1 && row_stride < vocab) || (draft_logits_dev && total > 1 && draft_row_stride < vocab))
    return record_failure(TABBY_EINVAL, "row strides must be at least vocab");
  const size_t size = dtype_size(dtype);
  if ((uintptr_t)logits_dev % size != 0 || (uintptr_t)draft_logits_dev % size != 0)
    return record_failure(TABBY_EINVAL, "logits must be aligned to their elements");
  if (((uintptr_t)drafts_dev | (uintptr_t)offsets_dev | (uintptr_t)tokens_dev | (uintptr_t)accepted_dev | (uintptr_t)status_dev) % 4 != 0 ||
      ((uintptr_t)uniforms_dev | (uintptr_t)params_dev) % 8 != 0)
    return record_failure(TABBY_EINVAL, "drafts, offsets and results must be 4-byte aligned, uniforms and params 8-byte");
  if (flags & ~TABBY_FLAG_FULL_VOCAB) return record_failure(TABBY_EINVAL, "unknown flags");
  int64_t need;
  rc = tabby_draft_workspace(requests, drafts_max, vocab, &need);
  if (rc) return rc;
  if ((uintptr_t)workspace_dev % 16 != 0 || workspace_bytes < need)
    return record_failure(TABBY_EINVAL, "workspace must be 16-byte aligned and hold " + std::to_string(need) + " bytes");
  const int slots = drafts_max + 1 + (draft_logits_dev ? drafts_max : 0);
  const int parts = verify_parts(rows + (draft_logits_dev ? total : 0), vocab);
  // Slots that no row fills take parts as well, which the workspace has to hold.
  const int fit = (int)std::max<int64_t>(1, std::min<int64_t>(parts, std::max<int64_t>((int64_t)requests * (2 * drafts_max + 1), kCus) / ((int64_t)requests * slots)));
  const int part_len = (int)((((int64_t)vocab + fit - 1) / fit + 31) / 32 * 32);
  const int used = (int)(((int64_t)vocab + part_len - 1) / part_len);
  const int segments = (vocab + kSegment - 1) / kSegment;
  const Space space = space_of(requests, slots, (int64_t)requests * slots * used, segments);
  char *w = (char *)workspace_dev;
  VerifyArgs a{logits_dev, draft_logits_dev, row_stride, draft_row_stride, drafts_dev, uniforms_dev, offsets_dev, params_dev,
               rows, requests, drafts_max, vocab, slots, (flags & TABBY_FLAG_FULL_VOCAB) != 0, used, part_len, segments,
               tokens_dev, accepted_dev, status_dev, (PartSum *)(w + space.sums), (uint64_t *)(w + space.entries),
               (RowDist *)(w + space.dists), (uint64_t *)(w + space.pools), (Decision *)(w + space.decisions),
               (double2 *)(w + space.segments)};
  // What is written lies apart from what is read.
  const RowSpan outputs[] = {row_span(tokens_dev, 1, (int64_t)requests * (drafts_max + 1), 0, 4), row_span(accepted_dev, 1, requests, 0, 4),
                             row_span(status_dev, 1, status_dev ? requests : 0, 0, 4), row_span(workspace_dev, 1, need, 0, 1)};
  const RowSpan logits = row_span(logits_dev, rows, vocab, row_stride, (int64_t)size);
  const RowSpan draft = row_span(draft_logits_dev, std::max<int64_t>(total, 1), vocab, draft_row_stride, (int64_t)size);
  for (const RowSpan &o : outputs) {
    if (!o.base || o.row_bytes == 0) continue;
    bool meets = rows_meet(logits, o.base, o.row_bytes) || (draft_logits_dev && total && rows_meet(draft, o.base, o.row_bytes)) ||
                 rows_meet(o, params_dev, (int64_t)requests * (int64_t)sizeof(tabby_row_params));
    if (total) meets |= rows_meet(o, drafts_dev, total * 4) || rows_meet(o, uniforms_dev, total * 8);
    if (offsets_dev) meets |= rows_meet(o, offsets_dev, ((int64_t)requests + 1) * 4);
    for (const RowSpan &other : outputs)
      if (&other != &o && other.base && other.row_bytes) meets |= rows_meet(o, other.base, other.row_bytes);
    if (meets) return record_failure(TABBY_EINVAL, "what a call writes must not overlap what it reads, nor each other");
  }
  const hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case TABBY_F32: return launch_verify<TABBY_F32>(a, s);
    case TABBY_F16: return launch_verify<TABBY_F16>(a, s);
    default: return launch_verify<TABBY_BF16>(a, s);
  }
}
