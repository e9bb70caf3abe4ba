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
//   decide  a workgroup to a request: its rows' parts together; how many tokens are accepted; pools are drawn from here. A
//           distribution is a maximum, a total and a threshold: an entry is in it if its (logit, index) is at or above that.
//           Of a whole vocabulary's that is cut, the parts' bins say between which bounds its probabilities lie: most
//           comparisons need no more
//   gather  (whole vocabularies that are cut) workgroups to a request: of the rows for which that is not enough, and of those
//           that the last token is drawn from, the entries among which the cut lies
//   settle  workgroups to a request: the exact cuts of these rows, then, by the last of them, the decision
//   weigh   (whole vocabularies) a workgroup to a segment of a deciding row: the sum of what is drawn from
//   pick    (whole vocabularies) a workgroup to a request: the draw, among segments, then within one
// Sums are in 64 bits, and exponentials within 5.5e-11: which token comes out hangs on comparisons of sums. Of whole
// vocabularies that are cut, running sums are compared with top_p of the total to within 1e-11 of it (2.5e-10 where there are more
// lists than have bins) and 2^-52 of the largest weight to an entry (3.4e-11 at 151,936 entries, 3.7e-9 at 2^24, at most); pools to the
// last bits.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>
#include <type_traits>

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
constexpr int kBlocksAimed = 512;
constexpr int kSharesMax = 32;
constexpr int kSegment = 1024;                // elements of a segment

enum Kind : int32_t { kInvalid = 0, kGreedy, kPool, kWhole };

// What `rows` leaves of a part.
struct PartSum {
  double sum;     // of exp((x - max) / T)
  float max;
  int32_t count;  // entries written
  int32_t bad;    // a NaN or +inf
  int32_t far;    // an entry so far above the reference that the bins do not hold it
  float reference;  // of the bins
};

// A row's distribution.
struct RowDist {
  double total;        // of the weights exp((x - max) / T) that are left
  double drafted;      // the drafted token's probability; below 0: there is no such token
  uint64_t threshold;  // the last entry's composite
  float max;
  int32_t count;       // a pool's entries that are left
  int32_t bad;         // a NaN, +inf, or nothing above -inf
  int32_t far;         // its bins do not hold all of it
};

// Where the cut of a whole vocabulary's distribution lies, as its row's bins tell.
struct RowCut {
  double from, total;  // the mass above the window; what top_p is a share of, or 0: not known. Both in units of 2^-shift.
  float least, most;   // the window: logits at or above `least` and below `most`
  int32_t shift;       // of the masses of its entries; 0: not known, and the window is all of the row
};

// What top_p of a row's total may be short of, relative to it, where that total is not the sum of the entries' own masses: from the
// bins, their polynomial's 2.5e-12 and its rounding's 1.9e-12, and as much for what lies above the window; from the parts' sums,
// up to three exponentials of 5.5e-11 each. Without it the last of the entries that make up the share exactly (nine of ten equal ones, for
// 0.9) would not do.
constexpr double kBinsOff = 1e-11, kSumsOff = 2.5e-10;

enum Draw : int32_t { kDone = 0, kFromTarget, kFromRest, kWithoutToken };

// What a request's last token is drawn from, where that is not a pool.
struct Decision {
  int64_t target, draft;         // the rows' first elements
  uint64_t threshold, draft_threshold;
  double inverse, of_target, of_draft;  // of the temperature and of the totals
  double uniform;
  float max, draft_max;
  int32_t draw, token;           // the token that is left out, or -1
  int64_t out;                   // its place among the tokens
};

// The rows of a request that have to be settled, by slots, and the workgroups that have settled theirs.
struct Needed {
  uint64_t slots[2];
  uint32_t settled;
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
  uint64_t *bins;        // [requests][slots][parts][kBins], or null
  uint64_t *pools;       // [requests][slots][kPoolMax], where a workgroup's LDS does not keep them
  Decision *decisions;   // [requests]
  double2 *segment_sums;  // [requests][segments]: of max(P - Q, 0) and of P
  RowCut *cuts;           // [requests][slots]
  Needed *needed;         // [requests]
  double2 *groups;        // [requests][slots][parts][64]: number and mass of the bins, 32 at a time
  uint32_t *gathered;     // [requests][slots][kSharesMax]: entries of the row's window, which lie where its bins did
  int shares;             // workgroups that gather a row
};

struct Setting {
  Kind kind;
  int k;
  double inverse, top_p;
  // Whether a whole vocabulary's distribution ends before its last entry.
  __device__ __forceinline__ bool cut(int vocab) const { return kind == kWhole && (top_p < 1.0 || k < vocab); }
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

// The parts that a row is cut into: what a wave holds of their lists has to fit.
constexpr int kWaveHeld = 1024;
struct Parts { int count, len; };
__device__ __forceinline__ Parts parts_of(const VerifyArgs &a, const Setting &set) {
  if (set.kind == kWhole || a.parts * set.k <= kWaveHeld) return {a.parts, a.part_len};
  const int most = kWaveHeld / set.k, len = ((a.vocab + most - 1) / most + 31) / 32 * 32;
  return {(a.vocab + len - 1) / len, len};
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

// The bins of a row whose distribution is cut: 16 to each power of two of exp((x - reference) / T), from 2^-96 to 2^32 on,
// each around its 2^(n/16). A bin holds the sum of its entries' weights in units of 2^(n/16) 2^-38, or their number and the
// sum in units of 2^(n/16) 2^-14: whole numbers, so that no order matters. The reference is the largest of 256 loads spread
// over the row, which all of its parts find alike.
constexpr int kPerOctave = 16, kBinsBelow = 96 * kPerOctave, kBinsAbove = kBins - kBinsBelow;
constexpr int kMassBits = 38, kSmallBits = 14, kCountShift = 39;
// All of a row in one bin: its number, and masses of at most 2^(1/32) < 33/32.
static_assert((uint64_t)kVerifyVocabMax <= UINT64_MAX / ((33ull << kMassBits) / 32 + 1) && (uint64_t)kVerifyVocabMax <= UINT64_MAX >> kCountShift &&
                  (uint64_t)kVerifyVocabMax <= ((1ull << kCountShift) - 1) / ((33ull << kSmallBits) / 32 + 1),
              "a bin's word holds them");

constexpr int kGroups = 64, kGroupBins = kBins / kGroups;  // the highest bins' group first

struct RowBins {
  double reference, scale;
  __device__ __forceinline__ RowBins(float reference_, const Setting &set) : reference(reference_), scale(set.inverse * (kPerOctave * 1.4426950408889634)) {}
  // In bins, above the reference's.
  __device__ __forceinline__ double height(float x) const { return ((double)x - reference) * scale; }
  // The bin of a height, no lower for a larger one, and what is left of it, in [-1/2, 1/2].
  static __device__ __forceinline__ int place(double height, double &f) {
    const double magic = 6755399441055744.0;  // as in exp_64
    const double shifted = height + magic;
    f = height - (shifted - magic);
    return (int)__builtin_bit_cast(uint32x2, shifted).x + kBinsBelow;
  }
  // For any logit: the lowest or the highest bin where they do not hold it.
  __device__ __forceinline__ int bin(float x) const {
    double f;
    return place(fmin(fmax(height(x), -(double)kBinsBelow), (double)(kBinsAbove - 1)), f);
  }
  // 2^(f/16) in units of 2^-38, rounded: the polynomial of degree 4 through it at the Chebyshev nodes, within 2.5e-12 of it,
  // plus 2^52, which leaves the whole number in the low bits.
  static __device__ __forceinline__ uint64_t mass(double f) {
    constexpr double kUnit = 274877906944.0;
    static_assert(kUnit == (double)(1ll << kMassBits), "the unit");
    double p = fma_const<true>(f, 1.4676387238435006e-07 * kUnit, 1.3551205154935067e-05 * kUnit);
    p = fma_const<true>(p, f, 0.0009383847926296646 * kUnit);
    p = fma_const<true>(p, f, 0.043321698760160544 * kUnit);
    return (uint64_t)__double_as_longlong(fma_const<true>(p, f, kUnit + 0x1p52)) & ((1ull << 52) - 1);
  }
  // What a bin holds: its number, if it has one, and its mass, relative to the reference's.
  static __device__ __forceinline__ double2 worth(uint64_t v, int bin, bool counts) {
    const double number = counts ? (double)(uint32_t)(v >> kCountShift) : 0.0;
    if (counts) v &= (1ull << kCountShift) - 1;
    static_assert(kPerOctave == 16 && kBinsBelow % kPerOctave == 0, "four bits of a bin are its sixteenths");
    double sixteenths = (bin & 8) != 0 ? 1.4142135623730951 : 1.0;
    sixteenths *= (bin & 4) != 0 ? 1.189207115002721 : 1.0;
    sixteenths *= (bin & 2) != 0 ? 1.0905077326652577 : 1.0;
    sixteenths *= (bin & 1) != 0 ? 1.0442737824274138 : 1.0;
    return {number, __builtin_ldexp((double)v * sixteenths, bin / kPerOctave - kBinsBelow / kPerOctave - (counts ? kSmallBits : kMassBits))};
  }
  // One entry and its mass, within 2^-14 of it.
  static __device__ __forceinline__ uint64_t one_and_mass(double f) {
    const float g = (float)f;
    const float w = __builtin_fmaf(__builtin_fmaf(g, 0.000938385f, 0.0433217f), g, 1.0f);
    return 1ull << kCountShift | (uint64_t)(uint32_t)(w * (float)(1 << kSmallBits) + 0.5f);
  }
};

template <int DT>
__device__ __forceinline__ float reference_of(const void *base, int vocab) {
  using E = Elem<DT>;
  const int loads = (vocab + E::kVec - 1) / E::kVec;
  u32x4 raw[4];
  int at[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    at[u] = (int)((int64_t)(u * 64 + wave_lane()) * loads >> 8) * E::kVec;
    raw[u] = load_values<DT, false>((const typename E::Bits *)base, at[u], vocab);
  }
  float top = -INFINITY;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    float v[E::kVec];
    E::widen16(raw[u], v);
#pragma unroll
    for (int j = 0; j < E::kVec; ++j) top = at[u] + j < vocab ? fmaxf(top, v[j]) : top;
  }
  top = wave_max(top);
  return top > -INFINITY && top < INFINITY ? top : 0.0f;
}

// A workgroup to a part of a row, 16 chunks of it on their way at once in eight waves. 16 x 9 rows of 128,000 f32 that are
// cut: 25 us, three parts to a row; of a workgroup's time 6.5 us do not depend on its length (the request's settings, the
// reference, the bins cleared and written), so that more parts take longer (eight: 37). 576 rows of 151,936 f32: 77 us, 4.6
// TB/s, of which the last 64 rows take the end for themselves; more copies of the bins against lanes that meet in
// one: slower, by their clearing.
template <int DT, int NW>
__global__ __launch_bounds__(NW * 64) void verify_rows_kernel(VerifyArgs a) {
  using Reader = PartReader<DT, false>;
  __shared__ union { ListScratch<NW> list; uint64_t bins[kBins]; } lds;
  ListScratch<NW> &scratch = lds.list;
  __shared__ double wave_sums[NW];
  __shared__ float wave_refs[NW], wave_tops[NW];
  const int row = (int)blockIdx.x / a.parts, part = (int)blockIdx.x - row * a.parts;
  const int request = row / a.slots, slot = row - request * a.slots;
  const int t = (int)threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const Setting set = setting_of(a, request);
  const SlotRow source = row_of<DT>(a, place_of(a, request), set.kind, slot);
  const Parts parts = parts_of(a, set);
  if (!source.used || part >= parts.count) return;
  const int begin = part * parts.len, len = min(parts.len, a.vocab - begin);
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
      if (t == 0) *out = PartSum{0.0, -INFINITY, 0, scratch.bad ? 1 : 0, 0, 0.0f};
      return;
    }
    const uint32_t need = min(n, (uint32_t)set.k);
    if (wave == 0) {
      const float m = wave_max(lane < NW ? wave_tops[lane] : -INFINITY);
      if (t == 0) *out = PartSum{0.0, m, (int)need, 0, 0, 0.0f};
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
  if (set.cut(a.vocab) && a.bins) {
    const RowBins bins(reference_of<DT>(source.base, a.vocab), set);
    const bool masses = set.k == a.vocab;  // else numbers as well
    for (int b = t; b < kBins; b += NW * 64) lds.bins[b] = 0;
    __syncthreads();
    bool far = false;
    if (c < reader.chunks) {
      do {
        bad |= !(top < INFINITY);
        far |= bins.height(top) > (double)(kBinsAbove - 1);
        largest = fmaxf(largest, top);
        // What is no number, or far, has no bin; nor has what lies beside a NaN, which hides it in `top`.
        if (__ballot(bad || far) != 0) continue;
        // Entries below the bins are no number of theirs, and far less than a sum tells: they count as the lowest bin's.
        if (masses) {
#pragma unroll
          for (int i = 0; i < kLane; ++i) {
            double f;
            const int at = bins.place(fmax(bins.height(x[i]), -(double)kBinsBelow), f);
            atomicAdd((unsigned long long *)&lds.bins[at], (unsigned long long)bins.mass(f));
          }
        } else {
#pragma unroll
          for (int i = 0; i < kLane; ++i) {
            double f;
            const int at = bins.place(fmax(bins.height(x[i]), -(double)kBinsBelow), f);
            atomicAdd((unsigned long long *)&lds.bins[at], (unsigned long long)bins.one_and_mass(f));
          }
        }
      } while (advance());
    }
    bad = __ballot(bad) != 0;
    far = __ballot(far) != 0;
    largest = wave_max(largest);
    if (lane == 0) wave_tops[wave] = bad ? INFINITY : largest;
    if (lane == 0) wave_refs[wave] = far ? 1.0f : 0.0f;
    __syncthreads();
    uint64_t *const to = a.bins + (int64_t)blockIdx.x * kBins;
    // A group of 32 bins lies in some neighbouring threads.
    constexpr int kPer = kBins / (NW * 64), kGroup = kGroupBins / kPer;
    double2 group{0.0, 0.0};
#pragma unroll 1
    for (int i = 0; i < kPer; ++i) {
      const int b = t * kPer + i;
      const uint64_t v = lds.bins[b];
      to[b] = v;
      const double2 w = RowBins::worth(v, b, !masses);
      group.x += w.x;
      group.y += w.y;
    }
#pragma unroll
    for (int d = 1; d < kGroup; d *= 2) {
      group.x += __shfl_xor(group.x, d);
      group.y += __shfl_xor(group.y, d);
    }
    if (t % kGroup == 0) a.groups[(int64_t)blockIdx.x * kGroups + (kGroups - 1 - t / kGroup)] = group;
    if (wave == 0) {
      const float m = wave_max(lane < NW ? wave_tops[lane] : -INFINITY);
      far = __ballot(lane < NW && wave_refs[lane] != 0.0f) != 0;
      if (t == 0) *out = m < INFINITY ? PartSum{0.0, m, 0, 0, far ? 1 : 0, (float)bins.reference} : PartSum{0.0, -INFINITY, 0, 1, 0, 0.0f};
    }
    return;
  }
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
    if (t == 0) *out = m < INFINITY ? PartSum{term, m, 0, 0, 0, 0.0f} : PartSum{0.0, -INFINITY, 0, 1, 0, 0.0f};
  }
}

// A whole row's distribution, not cut, from its parts; by a wave.
__device__ __forceinline__ RowDist whole_row(const VerifyArgs &a, int row, const Setting &set) {
  const int lane = wave_lane();
  const bool has = lane < a.parts;
  PartSum own{0.0, -INFINITY, 0, 0, 0, 0.0f};
  if (has) own = a.sums[(int64_t)row * a.parts + lane];
  const float m = wave_max(own.max);
  const bool bad = __ballot(own.bad) != 0 || !(m > -INFINITY);
  const bool far = __ballot(own.far) != 0;
  const double total = wave_sum(own.max > -INFINITY ? own.sum * exp_or_none(((double)own.max - (double)m) * set.inverse) : 0.0);
  return {total, 0.0, 0, m, 0, bad ? 1 : 0, far ? 1 : 0};
}

// A pool's weights run off by 1e-15 from the sampler's own exponential; a whole vocabulary's as its sums do.
__device__ __forceinline__ double weight_of(float x, float max, double inverse) {
  return exp_nonpos(((double)x - (double)max) * inverse);
}

// What a lane gets from another: CTRL and the rows of 16 lanes that it is for; 0 elsewhere.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T from_lane(T v) {
  static_assert(sizeof(T) == 4 || sizeof(T) == 8, "one or two registers");
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, ROWS == 0xF));
  } else {
    uint32x2 u = __builtin_bit_cast(uint32x2, v);
    u.x = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u.x, CTRL, ROWS, 0xF, ROWS == 0xF);
    u.y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u.y, CTRL, ROWS, 0xF, ROWS == 0xF);
    return __builtin_bit_cast(T, u);
  }
}

// Inclusive prefix sum over the wave's lanes, always in the same order (the steps of wave_inclusive_scan_u32).
template <typename T>
__device__ __forceinline__ T wave_prefix(T v) {
  v += from_lane<0x111, 0xF>(v);
  v += from_lane<0x112, 0xF>(v);
  v += from_lane<0x114, 0xF>(v);
  v += from_lane<0x118, 0xF>(v);
  v += from_lane<0x142, 0xA>(v);
  v += from_lane<0x143, 0xC>(v);
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

// Masses of a row's entries are whole multiples of 2^-shift: their sums are exact and do not depend on an order. As many bits as
// the sum of all of them, `total` times the largest at most, leaves of 61, and 51 at most, which the rounding below has
// room for: together they are off by 2^-52 of the largest to an entry, or by 2^-61 of the total where that is large.
__device__ __forceinline__ int mass_shift(double total) { return min(60 - ilogb(total), 51); }
__device__ __forceinline__ uint64_t mass_of(float x, float max, double inverse, double unit) {
  // At most 2^51: added to 2^52 it is rounded to a whole number, in the low bits.
  const double whole = __builtin_fma(exp_nonpos(((double)x - (double)max) * inverse), unit, 0x1p52);
  return (uint64_t)__double_as_longlong(whole) & ((1ull << 52) - 1);
}

// The smallest logit that lies in bin b or above, by a wave: 64 probes at a time among the keys.
__device__ __forceinline__ float bin_begin(const RowBins &bins, int b) {
  if (b >= kBins) return INFINITY;
  uint32_t low = kNegInfKey, high = key_of(INFINITY);  // low lies below, high does not
#pragma unroll 1
  while (high - low > 1) {
    const uint32_t step = (high - low + 63) / 64;
    const uint32_t probe = low + (uint32_t)(wave_lane() + 1) * step;
    const bool in = probe >= high || bins.bin(value_of(probe)) >= b;
    const int first = __builtin_ctzll(__ballot(in));  // the last lane's probe is high or beyond
    const uint32_t next_high = min(low + (uint32_t)(first + 1) * step, high);
    low += (uint32_t)first * step;
    high = next_high;
  }
  return value_of(high);
}

// A row's bins, its parts' together, by a wave: a lane to a group of them. Masses are relative to the reference's.
struct BinSums {
  const uint64_t *bins;  // [parts][kBins]
  int parts;
  bool counts;           // numbers and masses, else masses
  double count = 0.0, mass = 0.0, count_before, mass_before;  // the lane's, and what lies above
  double all_mass;

  __device__ __forceinline__ BinSums(const VerifyArgs &a, int row, bool counts_)
      : bins(a.bins + (int64_t)row * a.parts * kBins), parts(a.parts), counts(counts_) {
    const double2 *const groups = a.groups + (int64_t)row * a.parts * kGroups + wave_lane();
#pragma unroll 1
    for (int first = 0; first < parts; first += 4) {
      double2 v[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) v[p] = first + p < parts ? groups[(first + p) * kGroups] : double2{0.0, 0.0};
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        count += v[p].x;
        mass += v[p].y;
      }
    }
    count_before = wave_prefix(count);
    mass_before = wave_prefix(mass);
    all_mass = __shfl(mass_before, 63);
    count_before -= count;
    mass_before -= mass;
  }
  struct Found { int bin; double above, mass; };  // the mass above the bin, and its own
  // The highest bin at which the number (or the mass) from the highest on reaches `goal`; 0: there is none.
  __device__ __forceinline__ Found find(double goal, bool by_count) const {
    const double own = by_count ? count : mass, before = by_count ? count_before : mass_before;
    uint64_t who = __ballot(own > 0.0 && before + own >= goal);
    if (!who) return {0, 0.0, 0.0};
    const int owner = __builtin_ctzll(who);
    const double above = __shfl(mass_before, owner), above_own = __shfl(before, owner);
    // The owner's bins, a lane to each.
    const int b = kBins - kGroupBins * owner - 1 - (wave_lane() & (kGroupBins - 1));
    uint64_t v = 0;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) v += bins[(int64_t)p * kBins + b];
    double2 w = RowBins::worth(v, b, counts);
    if (wave_lane() >= kGroupBins) w = double2{0.0, 0.0};
    const double upto_mass = wave_prefix(w.y) + above, upto = by_count ? wave_prefix(w.x) + above_own : upto_mass;
    const bool some = (by_count ? w.x : w.y) > 0.0;
    who = __ballot(some && upto >= goal);
    // (By roundings none: the last that holds anything.)
    const int lane = who ? __builtin_ctzll(who) : 63 - __builtin_clzll(__ballot(some) | 1);
    return {__builtin_amdgcn_readlane(b, lane), __shfl(upto_mass - w.y, lane), __shfl(w.y, lane)};
  }
};

// What is known of a row whose distribution is cut, by a wave: its window, and the bounds of its drafted token's
// probability, x its logit. The distribution that is given lies between the bounds too.
__device__ __forceinline__ RowDist screen_row(const VerifyArgs &a, int row, const Setting &set, float x, RowCut &window, double &least_share,
                                              double &most_share) {
  RowDist dist = whole_row(a, row, set);
  const float m = dist.max;
  const bool by_count = set.k < a.vocab, by_mass = set.top_p < 1.0;
  int shift = dist.total > 0.0 ? mass_shift(dist.total) : 0;  // (with room for what the total is off by)
  window = {0.0, __builtin_ldexp(dist.total, shift), -INFINITY, INFINITY, shift};
  least_share = 0.0;
  most_share = INFINITY;
  if (dist.bad) return dist;
  const RowBins bins(a.sums[(int64_t)row * a.parts].reference, set);
  const double raised = bins.height(m);  // the row's maximum above the reference
  if (a.bins && !dist.far && raised > -256.0) {
    const BinSums sums(a, row, by_count);
    const double scale = exp2(raised * (-1.0 / kPerOctave));
    // What the sums may be off by: masses beside numbers are held in few bits.
    const double off = by_count ? 1e-4 : 1e-9, less = 1.0 - off, more = 1.0 + off;
    const double all = sums.all_mass;
    shift = mass_shift(all * scale * more);
    window.shift = shift;
    // The cut lies in the bins from `low` to `high`; `last` is the one of the k-th entry. (One loop: the code of one search.)
    BinSums::Found low{0, 0.0, 0.0}, high = low, last = low;
    double goal = by_count ? (double)set.k : set.top_p * all * (1.0 - kBinsOff);
#pragma unroll 1
    for (int search = 0; search < (by_count && by_mass ? 3 : 1); ++search) {
      const BinSums::Found found = sums.find(goal, by_count && search == 0);
      if (search == 0) last = high = low = found;
      else if (found.bin >= last.bin) (search == 1 ? low : high) = found;
      if (search == 0 && by_mass && by_count) goal = set.top_p * (last.above + last.mass) * more;
      if (search == 1) goal = set.top_p * last.above * less;
    }
    if (by_count && !by_mass) goal = last.above;
    if (by_count) window.least = bin_begin(bins, last.bin);
    if (low.bin > 0) {  // (the lowest bin holds what lies below it as well)
      const float least = bin_begin(bins, low.bin);
      if (!by_count) window = {__builtin_ldexp(high.above * scale, shift), __builtin_ldexp(all * scale, shift), least, bin_begin(bins, high.bin + 1), shift};
      const double total_least = fmax(high.above, goal) * scale * less, total_most = (low.above + low.mass) * scale * more;
      dist.total = 0.5 * (total_least + total_most);
      dist.threshold = (uint64_t)key_of(least) << 32;
      if (!(x > -INFINITY)) {
        most_share = 0.0;
      } else {
        const int b = bins.bin(x);
        const double w = exp_or_none(((double)x - (double)m) * set.inverse);
        if (b > high.bin) least_share = w / total_most * (1.0 - 1e-9);
        most_share = b < low.bin ? 0.0 : w / total_least * (1.0 + 1e-9);
      }
      return dist;
    }
    window = {0.0, 0.0, -INFINITY, INFINITY, shift};
  } else if (!by_count && window.total > 0.0) {
    // Entries below (1 - top_p) total / vocab hold less than 1 - top_p together. (A margin for roundings.)
    const double low = (1.0 - set.top_p) * dist.total / (double)a.vocab * (1.0 - 1e-6);
    const double bound = (double)m - fmax(-log(low), 0.0) / set.inverse - fabs((double)m) * 1e-6;
    window.least = bound > -3.4e38 ? (float)bound : -INFINITY;
  }
  return dist;
}

// A wave's work on a row whose distribution is a list: its parts' entries together in `held`, those at or above a
// bound ranked by counting, and cut. The entries that are left go to `pool`, in order.
__device__ __forceinline__ RowDist pool_row(const VerifyArgs &a, int row, const Setting &set, uint64_t *held, uint64_t *pool) {
  const int lane = wave_lane();
  const int parts = parts_of(a, set).count;
  const PartSum *sums = a.sums + (int64_t)row * a.parts;
  const uint64_t *entries = a.entries + (int64_t)row * a.parts * kPoolMax;
  // A lane to a part.
  PartSum own{0.0, -INFINITY, 0, 0, 0, 0.0f};
  if (lane < parts) own = sums[lane];
  const float m = wave_max(own.max);
  RowDist dist{0.0, 0.0, 0, m, 0, 0, 0};
  dist.bad = __ballot(own.bad) != 0 || !(m > -INFINITY);
  if (dist.bad) return dist;
  // The parts' entries one after another, a part's turned by five places from the one before: each of the 64 lanes' four
  // columns has entries of different ranks.
  const int slots = parts * set.k;
  const float per = 1.0f / (float)set.k;  // slots <= 2^10: (i + 1/2) / k has bits to spare
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll 1
  for (int first = 0; first < slots; first += 8 * 64) {
    uint64_t e[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = first + u * 64 + lane, p = (int)(((float)i + 0.5f) * per), turned = i - p * set.k + 5 * p;
      const int at = turned - (int)(((float)turned + 0.5f) * per) * set.k;
      // By all lanes: what a lane that is switched off holds is not read.
      const int listed = __builtin_amdgcn_ds_bpermute((p & 63) << 2, own.count);
      e[u] = i < slots && at < listed ? entries[p * kPoolMax + at] : 0;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (first + u * 64 + lane < slots) held[first + u * 64 + lane] = e[u];
      v[u & 3] = max(v[u & 3], composite_key(e[u]));
    }
  }
  uint32_t theta = 0;
  if (parts > 1) {
    uint32_t all[1] = {max(max(v[0], v[1]), max(v[2], v[3]))};
    theta = set.k <= 32 ? kth_largest<1>(all, set.k) : kth_largest<4>(v, set.k);
  }
  wave_lds_sync();
  uint32_t n = 0;
#pragma unroll 1
  for (int first = 0; first < slots; first += 64) {
    // To the front: what is written was read before.
    const uint64_t e = first + lane < slots ? held[first + lane] : 0;
    const bool in = e != 0 && composite_key(e) >= theta;
    const uint64_t who = __ballot(in);
    if (in) held[n + lanes_before(who)] = e;
    n += (uint32_t)__popcll(who);
    wave_lds_sync();
  }
  const uint32_t need = min(n, (uint32_t)set.k);
#pragma unroll 1
  for (uint32_t i = (uint32_t)lane; i < n; i += 64) {
    const uint64_t e = held[i];
    uint32_t rank = 0;
#pragma unroll 4
    for (uint32_t j = 0; j < n; ++j) rank += held[j] > e ? 1u : 0u;
    if (rank < need) pool[rank] = e;
  }
  wave_lds_sync();
  double sum[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t i = (uint32_t)(lane + 64 * h);
    const double w = i >= need ? 0.0 : set.kind == kGreedy ? 1.0 : weight_of(value_of(composite_key(pool[i])), m, set.inverse);
    sum[h] = wave_prefix(w);
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
  return dist;
}

// The probability of a row's drafted token, x its logit.
__device__ __forceinline__ double share_of(const RowDist &d, const Setting &set, int token, int vocab, float x) {
  if (token < 0 || token >= vocab) return -1.0;
  if (!(x > -INFINITY) || composite(key_of(x), (uint32_t)token) < d.threshold) return 0.0;
  return (set.kind == kGreedy ? 1.0 : weight_of(x, d.max, set.inverse)) / d.total;
}

// How many of a request's tokens are accepted, by its workgroup, whose first wave compares.
struct Verdict { int accepted, status; };
__device__ __forceinline__ Verdict verdict_of(const VerifyArgs &a, int request, const Setting &set, const Place &place, const RowDist *dists, Verdict &shared) {
  const int t = (int)threadIdx.x, first_draft = a.drafts_max + 1;
  const bool drawn = a.draft_logits != nullptr && set.kind != kGreedy;  // else the drafted tokens were certain
  if (t < 64) {
    const bool asked = place.drafts >= 0 && t < place.drafts && set.kind != kInvalid;
    bool good = false, broken = false, unknown = false;
    if (asked) {
      const double share = dists[t].drafted, claim = drawn ? dists[first_draft + t].drafted : 1.0;
      broken = dists[t].bad || (drawn && dists[first_draft + t].bad);
      unknown = !broken && share < 0.0;
      good = !broken && !unknown && a.uniforms[place.first_draft + t] * claim < share;
    }
    const uint64_t goods = __ballot(good), brokens = __ballot(broken), unknowns = __ballot(unknown);
    if (t == 0) {
      int n = 0, status = TABBY_EINVAL;
      if (place.drafts >= 0 && set.kind != kInvalid) {
        n = min((int)__builtin_ctzll(~goods), place.drafts);  // lane 63 never has a token
        const uint64_t here = 1ull << n;
        status = (brokens & here) || (n == place.drafts && dists[n].bad) ? TABBY_EDOMAIN : (unknowns & here) ? TABBY_EINVAL : TABBY_OK;
      }
      shared = {n, status};
    }
  }
  __syncthreads();
  const int n = shared.accepted, status = shared.status;
  int32_t *tokens = a.tokens + (int64_t)request * (a.drafts_max + 1);
  if (t <= a.drafts_max && (status != TABBY_OK || t != n)) tokens[t] = status == TABBY_OK && t < n ? a.drafts[place.first_draft + t] : -1;
  if (t == 0) {
    a.accepted[request] = status == TABBY_OK ? n : 0;
    if (a.status) a.status[request] = status;
  }
  return {n, status};
}

__device__ __forceinline__ Draw draw_of(const VerifyArgs &a, const Setting &set, const Place &place, int accepted) {
  if (accepted >= place.drafts || set.kind == kGreedy) return kFromTarget;
  return a.draft_logits ? kFromRest : kWithoutToken;
}

// What the last token of a whole vocabulary is drawn from.
__device__ __forceinline__ Decision decision_of(const VerifyArgs &a, int request, const Setting &set, const Place &place, const RowDist *dists, Verdict v) {
  const int n = v.accepted, first_draft = a.drafts_max + 1;
  if (v.status != TABBY_OK || set.kind != kWhole) return Decision{};
  const Draw draw = draw_of(a, set, place, n);
  const RowDist &p = dists[n], &q = dists[draw == kFromRest ? first_draft + n : n];
  return {(int64_t)(place.first + n) * a.stride, (int64_t)(place.first_draft + n) * a.draft_stride,
          p.threshold, q.threshold, set.inverse, 1.0 / p.total, 1.0 / q.total, a.params[request].uniform, p.max, q.max, draw,
          draw == kWithoutToken ? a.drafts[place.first_draft + n] : -1, (int64_t)request * (a.drafts_max + 1) + n};
}

// Which rows have to be settled, by the first wave, from the bounds of the drafted tokens' probabilities: [slot][least, most].
// Up to the first token that is refused for certain, both rows of each that is neither refused nor accepted for certain, and
// the rows that the last token is drawn from then.
__device__ __forceinline__ Needed needed_of(const VerifyArgs &a, const Place &place, const RowDist *dists, const double (*bounds)[2]) {
  const int lane = wave_lane(), first_draft = a.drafts_max + 1;
  const bool drawn = a.draft_logits != nullptr, asked = lane < place.drafts;
  bool stops = false, refused = false, open = false;
  if (asked) {
    const double u = a.uniforms[place.first_draft + lane];
    const double claim_least = drawn ? bounds[first_draft + lane][0] : 1.0, claim_most = drawn ? bounds[first_draft + lane][1] : 1.0;
    stops = dists[lane].bad || (drawn && dists[first_draft + lane].bad) || dists[lane].drafted < 0.0;
    const bool plain = u >= 0.0 && u <= 1.0;
    refused = !stops && plain && !(u * claim_least < bounds[lane][1]);
    open = !stops && !refused && !(plain && u * claim_most < bounds[lane][0]);
  }
  const uint64_t ends = __ballot(stops || refused), refusals = __ballot(refused), opens = __ballot(open);
  const int last = ends ? __builtin_ctzll(ends) : place.drafts;  // at most 63
  uint64_t target = opens & ((1ull << last) - 1), draft = drawn ? target : 0;
  if (last == place.drafts) {
    if (!dists[last].bad) target |= 1ull << last;
  } else if (refusals >> last & 1) {
    target |= 1ull << last;
    if (drawn) draft |= 1ull << last;
  }
  Needed needed{{target, 0}, 0};
  needed.slots[0] |= first_draft < 64 ? draft << first_draft : 0;
  needed.slots[1] = first_draft < 64 ? draft >> 1 >> (63 - first_draft) : draft << (first_draft - 64);
  return needed;
}

// A workgroup of NW waves to a request: a wave to a row gives its distribution and the probability of its drafted token;
// then the first refusal; then, for pools, the draw. A chain of latencies: of 12.5 us for nine rows of ten lists of 40 each,
// the lists' entries take 3, their bound 2, compaction and ranks 2, the wait for the other rows 3, the draw 2. Rows that are
// cut take their bounds here (16 requests of nine rows: 12 us), which spares the settling of seven rows in nine.
template <int DT, int NW, bool FULL>
__global__ __launch_bounds__(NW * 64) void verify_decide_kernel(VerifyArgs a) {
  using E = Elem<DT>;
  constexpr int kKept = NW;  // rows whose entries stay in LDS
  __shared__ uint64_t held[NW][kWaveHeld], pools[kKept][kPoolMax];
  __shared__ RowDist dists[2 * kDraftsMax + 1];
  __shared__ double rest[kPoolMax], all[kPoolMax];
  __shared__ double bounds[FULL ? 2 * kDraftsMax + 1 : 1][2];
  __shared__ Verdict shared;
  __shared__ bool waits;
  __shared__ uint32_t ids[kPoolMax];
  const int request = (int)blockIdx.x, t = (int)threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const Setting set = setting_of(a, request);
  const Place place = place_of(a, request);
  for (int slot = wave; slot < a.slots; slot += NW) {
    const SlotRow source = row_of<DT>(a, place, set.kind, slot);
    if (!source.used) continue;
    // The drafted token's logit, on its way while the row's parts are.
    int token = -1;
    float x = -INFINITY;
    if (source.drafted >= 0) {
      token = a.drafts[source.drafted];
      if (token >= 0 && token < a.vocab) x = E::widen(((const typename E::Bits *)source.base)[token]);
    }
    const int row = request * a.slots + slot;
    RowDist d;
    if (!FULL || set.kind != kWhole) {
      d = pool_row(a, row, set, held[wave], pools[a.slots > kKept ? wave : slot]);
    } else if (!set.cut(a.vocab)) {
      d = whole_row(a, row, set);
    } else {
      RowCut window;
      double least, most;
      d = screen_row(a, row, set, x, window, least, most);
      if (lane == 0) {
        bounds[slot][0] = least;
        bounds[slot][1] = most;
        a.cuts[row] = window;
      }
    }
    if (source.drafted >= 0 && !d.bad) d.drafted = share_of(d, set, token, a.vocab, x);
    if (FULL && lane == 0) a.dists[row] = d;
    if (lane == 0) dists[slot] = d;
    if (set.kind == kPool && a.slots > kKept) {
      for (int i = lane; i < d.count; i += 64) a.pools[(int64_t)row * kPoolMax + i] = pools[wave][i];
    }
  }
  __syncthreads();
  if constexpr (FULL) {
    if (wave == 0) {
      Needed needed{};
      if (place.drafts >= 0 && set.cut(a.vocab)) needed = needed_of(a, place, dists, bounds);
      if (t == 0) {
        a.needed[request] = needed;
        waits = (needed.slots[0] | needed.slots[1]) != 0;
        if (waits) a.decisions[request] = Decision{};
      }
    }
    __syncthreads();
    if (waits) return;
  }
  const int first_draft = a.drafts_max + 1;  // slot of the draft's rows
  const Verdict verdict = verdict_of(a, request, set, place, dists, shared);
  const int n = verdict.accepted, status = verdict.status;
  int32_t *tokens = a.tokens + (int64_t)request * (a.drafts_max + 1);
  if (FULL && t == 0) a.decisions[request] = decision_of(a, request, set, place, dists, verdict);
  if (status != TABBY_OK || set.kind == kWhole) return;
  // A pool: what is left of the target's entries, in the vocabulary's order.
  const Draw draw = draw_of(a, set, place, n);
  const RowDist p = dists[n], q = draw == kFromRest ? dists[first_draft + n] : p;
  if (set.kind == kGreedy) {
    if (t == 0) tokens[n] = (int32_t)composite_index(p.threshold);
    return;
  }
  uint64_t *target = pools[n % kKept], *draft = pools[(first_draft + n) % kKept];
  if (a.slots > kKept) {
    // More rows than LDS keeps.
    target = held[0];
    draft = held[1];
    const int64_t at = (int64_t)request * a.slots;
    if (t < p.count) target[t] = a.pools[(at + n) * kPoolMax + t];
    if (draw == kFromRest && t < q.count) draft[t] = a.pools[(at + first_draft + n) * kPoolMax + t];
    __syncthreads();
  }
  // Some threads to an entry: how many tokens come before its own, and what the draft takes of it.
  constexpr int kShare = NW * 64 / kPoolMax;
  const int i = t / kShare, part = t % kShare;
  if (i < p.count) {
    const uint64_t own = target[i];
    const uint32_t id = composite_index(own);
    uint32_t before = 0, found = 0;  // the place in the draft's list, from 1
#pragma unroll 1
    for (int j = part; j < p.count; j += kShare) before += composite_index(target[j]) < id ? 1u : 0u;
    if (draw == kFromRest) {
#pragma unroll 1
      for (int j = part; j < q.count; j += kShare)
        if (composite_index(draft[j]) == id) found = (uint32_t)j + 1;
    }
#pragma unroll
    for (int stride = 1; stride < kShare; stride *= 2) {
      before += xor_lane_by(before, stride);
      found = max(found, xor_lane_by(found, stride));
    }
    if (part == 0) {
      const double share = weight_of(value_of(composite_key(own)), p.max, set.inverse) / p.total;
      double left = share;
      if (found) left = fmax(share - weight_of(value_of(composite_key(draft[found - 1])), q.max, set.inverse) / q.total, 0.0);
      if (draw == kWithoutToken && (int)id == a.drafts[place.first_draft + n]) left = 0.0;
      rest[before] = left;
      all[before] = share;
      ids[before] = id;
    }
  }
  __syncthreads();
  if (wave != 0) return;
  // The first whose running sum exceeds the share; the last with a weight where none does.
  double w[2], sum[2], total = 0.0;
#pragma unroll 1
  for (int tries = 0; tries < 2; ++tries) {
    const double *const of = tries == 0 ? rest : all;  // nothing left: P is Q, but for roundings
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w[h] = lane + 64 * h < p.count ? of[lane + 64 * h] : 0.0;
      sum[h] = wave_prefix(w[h]);
    }
    sum[1] += __shfl(sum[0], 63);
    total = __shfl(sum[1], 63);
    if (total > 0.0) break;
  }
  const double goal = a.params[request].uniform * total;
  const uint64_t over[2] = {__ballot(w[0] > 0.0 && sum[0] > goal), __ballot(w[1] > 0.0 && sum[1] > goal)};
  const uint64_t some[2] = {__ballot(w[0] > 0.0), __ballot(w[1] > 0.0)};
  int at = 0;
  if (over[0]) at = __builtin_ctzll(over[0]);
  else if (over[1]) at = 64 + __builtin_ctzll(over[1]);
  else if (some[1]) at = 127 - __builtin_clzll(some[1]);
  else if (some[0]) at = 63 - __builtin_clzll(some[0]);
  if (lane == 0) tokens[n] = (int32_t)ids[at];
}

constexpr int kSettleWaves = 8;
constexpr int kSettleThreads = kSettleWaves * 64;
constexpr int kHeldMax = 64;          // entries that are ranked at once, by a wave
constexpr int kCells = kSettleThreads;
constexpr int kCandidatesMax = 5632;  // entries of a row's window, in LDS

struct SettleScratch {
  uint64_t candidates[kCandidatesMax];
  uint64_t masses[kCells];
  uint32_t counts[kCells];
  RowDist dists[2 * kDraftsMax + 1];
  uint64_t held[kHeldMax], sorted[kHeldMax];
  uint64_t wave64[kSettleWaves], wave64_mass[kSettleWaves];
  uint64_t found_measure, found_mass, found_entry;
  uint32_t found_bin, taken, gathered, begins[kSharesMax + 1];
  Verdict shared;
  bool last;
};

// The entries of a row at or above `least` (and above -inf) and below `most`, by the whole workgroup. They are gathered in LDS
// first, so that what is done with them is done by full waves.
template <int DT>
struct Candidates {
  using E = Elem<DT>;
  using Bits = typename E::Bits;
  static constexpr int kLoad = kSettleThreads * E::kVec;  // elements of a load
  static_assert(kLoad <= kCandidatesMax, "a load's entries find room");
  const Bits *row;
  int vocab;
  float least, most;
  SettleScratch &s;
  bool resident = false;  // all of them lie in s.candidates, s.gathered of them

  __device__ __forceinline__ Candidates(const void *base, int vocab_, const RowCut &window, SettleScratch &s_)
      : row((const Bits *)base), vocab(vocab_), least(window.least), most(window.most), s(s_) {}
  __device__ __forceinline__ int place(int load) const { return load * kLoad + (int)threadIdx.x * E::kVec; }
  __device__ __forceinline__ int loads() const { return (vocab + kLoad - 1) / kLoad; }
  __device__ __forceinline__ u32x4 read(int load) const {
    const int at = place(load);
    return at < vocab ? load_values<DT, false>(row, at, vocab) : u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ bool in(float v, int e) const { return e < vocab && v >= least && v < most && v > -INFINITY; }
  // The entries of a load behind those that are there already.
  __device__ __forceinline__ void append(u32x4 raw, int load) const {
    float v[E::kVec];
    E::widen16(raw, v);
    const int at = place(load);
    uint32_t own = 0;
#pragma unroll
    for (int j = 0; j < E::kVec; ++j) own += in(v[j], at + j) ? 1u : 0u;
    if (!__ballot(own != 0)) return;
    const uint32_t upto = wave_inclusive_scan_u32(own);
    uint32_t to = 0;
    if (wave_lane() == 63) to = atomicAdd(&s.gathered, upto);
    to = (uint32_t)__builtin_amdgcn_readlane((int)to, 63) + upto - own;
#pragma unroll
    for (int j = 0; j < E::kVec; ++j) {
      if (!in(v[j], at + j)) continue;
      if (to < (uint32_t)kCandidatesMax) s.candidates[to] = composite(key_of(v[j]), (uint32_t)(at + j));
      ++to;
    }
  }
  // All of them, if they are as few as LDS holds.
  __device__ __forceinline__ void fill() {
    constexpr int kAhead = 4;
    __syncthreads();
    if (threadIdx.x == 0) s.gathered = 0;
    u32x4 raw[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) raw[u] = read(u);
    __syncthreads();
#pragma unroll 1
    for (int first = 0; first < loads(); first += kAhead) {
      u32x4 next[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) next[u] = read(first + kAhead + u);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) append(raw[u], first + u);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) raw[u] = next[u];
    }
    __syncthreads();
    resident = s.gathered <= (uint32_t)kCandidatesMax;
  }
  // Those that were gathered, if they all were and are as few as LDS holds.
  __device__ __forceinline__ void take(const uint64_t *list, const uint32_t *counts, int shares, uint32_t room) {
    static_assert(kSharesMax * 16 == kSettleThreads, "sixteen threads to a share");
    const int share = (int)threadIdx.x >> 4;
    __syncthreads();
    if (threadIdx.x < 64) {
      const uint32_t own = (int)threadIdx.x < shares ? counts[threadIdx.x] : 0, upto = wave_inclusive_scan_u32(own);
      if (threadIdx.x < kSharesMax) s.begins[threadIdx.x] = upto - own;
      const bool fits = __ballot(own > room) == 0;
      if (threadIdx.x == 63) s.gathered = fits ? upto : ~0u;
      if (threadIdx.x == kSharesMax - 1) s.begins[kSharesMax] = upto;
    }
    __syncthreads();
    resident = s.gathered <= (uint32_t)kCandidatesMax;
    if (resident) {
      const uint32_t begin = s.begins[share], n = s.begins[share + 1] - begin;
      for (uint32_t i = threadIdx.x & 15; i < n; i += 16) s.candidates[begin + i] = list[(int64_t)share * room + i];
    }
    __syncthreads();
  }
  // f(logit, composite) of every one of them. More than LDS holds: the row again, as much of it as fits at a time. (One request over
  // 151,936 f32: 54 us with top_k 5,000, 352 with 6,000, 668 with 100,000; a constant row, whose entries all meet in a cell or
  // two, 1.6 ms, and 153 ms at 2^24.)
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    const int all = resident ? 1 : loads();
    if (!resident) {
      __syncthreads();
      if (threadIdx.x == 0) s.gathered = 0;
      __syncthreads();
    }
#pragma unroll 1
    for (int load = 0; load < all; ++load) {
      if (!resident) append(read(load), load);
      __syncthreads();
      const uint32_t n = s.gathered;
      const bool full = load + 1 == all || n + (uint32_t)kLoad > (uint32_t)kCandidatesMax;
      if (full) {
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < n; i += kSettleThreads) f(value_of(composite_key(s.candidates[i])), s.candidates[i]);
      }
      __syncthreads();
      if (full && !resident) {
        if (threadIdx.x == 0) s.gathered = 0;
        __syncthreads();
      }
    }
  }
};

// The cut of a row, exactly: after the k-th entry, and where top_p is reached. It lies in a cell of composites, which is
// narrowed by the counts and masses of 512 equal parts of it until it holds as few as a wave ranks.
template <int DT>
__device__ __forceinline__ void settle_row(const VerifyArgs &a, const Setting &set, const RowCut &window, const Candidates<DT> &left, RowDist &dist, SettleScratch &s) {
  const int t = (int)threadIdx.x;
  const float m = dist.max;
  int shift = window.shift;
  if (shift == 0) {
    // Their sum first, in the masses that as many entries alike would leave.
    const double coarse = __builtin_ldexp(1.0, mass_shift((double)a.vocab));
    uint64_t sum = 0, all;
    left.each([&](float x, uint64_t) { sum += mass_of(x, m, set.inverse, coarse); });
    block_prefix<kSettleWaves>(sum, s.wave64, all);
    shift = mass_shift(((double)all + (double)a.vocab) / coarse);
  }
  const double unit = __builtin_ldexp(1.0, shift);
  const bool by_count = set.k < a.vocab, by_mass = set.top_p < 1.0;
  double total = window.total;  // of what top_p is a share of, in units; 0: not known
  uint64_t goal = 0, entry = 0, left_mass = 0;  // the last entry that is left; of what is left
  // The smallest whole number of units that is top_p of the total, within what that may be off by, or the rounding of the
  // masses where it is their own sum (so that 900 of 1,000 equal entries are 0.9 of them); at least one.
  const double off = by_count || !(window.total > 0.0) ? 1e-12 : a.bins ? kBinsOff : kSumsOff;
  auto aim = [&]() { goal = (uint64_t)fmax(ceil(set.top_p * total * (1.0 - off - 1.0 / unit)), 1.0); };
#pragma unroll 1
  for (int stage = by_count ? 0 : 1; stage < (by_mass ? 2 : 1); ++stage) {
    const bool masses = stage == 1;
    // The cell: from low to high.
    uint64_t low = masses && by_count ? entry : window.least > -INFINITY ? (uint64_t)key_of(window.least) << 32 : 0;
    uint64_t high = ((uint64_t)key_of(fminf(m, window.most)) << 32 | 0xffffffffu) - (window.most <= m ? 1ull << 32 : 0);
    uint64_t above_mass = masses && !by_count ? (uint64_t)(window.from + 0.5) : 0, above = above_mass;  // what lies above it
    if (!masses) goal = (uint64_t)set.k;
    else if (total > 0.0) aim();
    uint32_t in_cell = left.resident && (!masses || total > 0.0) && !(masses && by_count) ? s.gathered : ~0u;
    // (A cell of one composite holds one entry. One whose masses are all zero ends the search with none.)
#pragma unroll 1
    while (in_cell > (uint32_t)kHeldMax) {
      const int shift = max(55 - (int)__clzll(high - low), 0);
      static_assert(kCells == 512, "nine bits");
      s.counts[t] = 0;
      s.masses[t] = 0;
      if (t == 0) {
        s.found_bin = s.taken = 0;
        s.found_measure = s.found_mass = 0;
      }
      __syncthreads();
      left.each([&](float x, uint64_t c) {
        if (c < low || c > high) return;
        const uint32_t to = (uint32_t)((c - low) >> shift);
        atomicAdd(&s.counts[to], 1u);
        atomicAdd((unsigned long long *)&s.masses[to], (unsigned long long)mass_of(x, m, set.inverse, unit));
      });
      // The highest part at which the running count (or mass) from the highest on reaches the goal -- where none does, the
      // lowest that holds anything.
      const int cell = kCells - 1 - t;
      const uint64_t mass = s.masses[cell], own = masses ? mass : s.counts[cell];
      uint64_t all, all_mass;
      const uint64_t before = block_prefix<kSettleWaves>(own, s.wave64, all) - own;
      const uint64_t before_mass = masses ? before : block_prefix<kSettleWaves>(mass, s.wave64_mass, all_mass) - mass;
      if (masses && !(total > 0.0)) {
        // The first time, with all of the row in the cell.
        total = (double)all;
        aim();
      }
      const uint64_t want = goal <= above ? 1 : goal - above < all ? goal - above : all;
      if (own > 0 && before < want && before + own >= want) {
        s.found_bin = (uint32_t)cell;
        s.found_measure = before;
        s.found_mass = before_mass;
        s.taken = s.counts[cell];
      }
      __syncthreads();
      above += s.found_measure;
      above_mass += s.found_mass;
      in_cell = s.taken;
      low += (uint64_t)s.found_bin << shift;
      const uint64_t end = low + ((1ull << shift) - 1);
      high = end < high ? end : high;
      __syncthreads();
    }
    __syncthreads();
    if (t == 0) s.taken = 0;
    __syncthreads();
    left.each([&](float, uint64_t c) {
      if (c < low || c > high || in_cell == 0) return;
      const uint32_t at = atomicAdd(&s.taken, 1u);
      if (at < (uint32_t)kHeldMax) s.held[at] = c;
    });
    // In order: the first that reaches the goal, or the last there is.
    if (t < 64) {
      const uint32_t n = min(s.taken, (uint32_t)kHeldMax);
      const uint64_t own = (uint32_t)t < n ? s.held[t] : 0;
      uint32_t rank = 0;
#pragma unroll 4
      for (uint32_t j = 0; j < n; ++j) rank += s.held[j] > own ? 1u : 0u;
      if ((uint32_t)t < n) s.sorted[rank] = own;
      wave_lds_sync();
      const uint64_t mine = (uint32_t)t < n ? s.sorted[t] : 0;
      const uint64_t mass = (uint32_t)t < n ? mass_of(value_of(composite_key(mine)), m, set.inverse, unit) : 0;
      const uint64_t upto = wave_prefix(mass) + above_mass;
      // (Of masses, `above` is above_mass.)
      const uint64_t who = __ballot((uint32_t)t < n && (masses ? upto >= goal : above + (uint64_t)t + 1 >= goal));
      const int at = who ? __builtin_ctzll(who) : (int)max(n, 1u) - 1;
      if (t == at) {
        s.found_entry = n ? mine : low;
        s.found_mass = upto;
      }
    }
    __syncthreads();
    entry = s.found_entry;
    left_mass = s.found_mass;
    total = (double)left_mass;
    __syncthreads();
  }
  dist.threshold = entry;
  dist.total = (double)left_mass / unit;
}

// f(slot) of the rows that have to be settled, from the `first` on, every `step`-th.
template <class F>
__device__ __forceinline__ void each_needed(const Needed &needed, int first, int step, F f) {
  int n = 0;
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
#pragma unroll 1
    for (uint64_t rest = needed.slots[h]; rest; rest &= rest - 1, ++n)
      if (n % step == first) f(h * 64 + (int)__builtin_ctzll(rest));
  }
}

// The entries that a share of a row's gathering has room for: they lie where its bins did.
__device__ __forceinline__ uint32_t share_room(const VerifyArgs &a) { return (uint32_t)(a.parts * kBins / a.shares); }

// A row's entries in its window, to the row's lists, a workgroup to a share: loads far apart, so that no order of the
// vocabulary fills one of them. (One workgroup to a row passes over it at 25 GB/s: 20 us for 128,000 f32; 32 take 7. The last
// of them going on to settle the row instead of a launch of its own: 41 us against 20, for the order it asks of memory.)
constexpr int kGatherThreads = 256;
constexpr int kGatherRows = 2;  // of a request, at a time
constexpr int kGatherBlocks = 2048;
constexpr int kSettleRows = 4;
template <int DT>
__global__ __launch_bounds__(kGatherThreads) void verify_gather_kernel(VerifyArgs a) {
  using E = Elem<DT>;
  using Bits = typename E::Bits;
  __shared__ uint32_t gathered;
  const int share = (int)blockIdx.x, request = (int)blockIdx.y, t = (int)threadIdx.x;
  const Needed needed = a.needed[request];
  const Place place = place_of(a, request);  // (on its way beside the line above)
  if (!(needed.slots[0] | needed.slots[1])) return;
  const uint32_t room = share_room(a);
  each_needed(needed, (int)blockIdx.z, kGatherRows, [&](int slot) {
    const int row = request * a.slots + slot;
    const RowCut window = a.cuts[row];
    const Bits *const base = (const Bits *)row_of<DT>(a, place, kWhole, slot).base;
    uint64_t *const list = a.bins + (int64_t)row * a.parts * kBins + (int64_t)share * room;
    __syncthreads();
    if (t == 0) gathered = 0;
    __syncthreads();
    constexpr int kAhead = 4, kLoad = kGatherThreads * E::kVec;
    const int loads = (a.vocab + kLoad - 1) / kLoad;
#pragma unroll 1
    for (int first = share; first < loads; first += kAhead * a.shares) {
      u32x4 raw[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int at = (first + u * a.shares) * kLoad + t * E::kVec;
        raw[u] = at < a.vocab ? load_values<DT, false>(base, at, a.vocab) : u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int at = (first + u * a.shares) * kLoad + t * E::kVec;
        float v[E::kVec];
        E::widen16(raw[u], v);
        uint32_t own = 0;
        bool in[E::kVec];
#pragma unroll
        for (int j = 0; j < E::kVec; ++j) {
          in[j] = at + j < a.vocab && v[j] >= window.least && v[j] < window.most && v[j] > -INFINITY;
          own += in[j] ? 1u : 0u;
        }
        if (!__ballot(own != 0)) continue;
        const uint32_t upto = wave_inclusive_scan_u32(own);
        uint32_t to = 0;
        if (wave_lane() == 63) to = atomicAdd(&gathered, upto);
        to = (uint32_t)__builtin_amdgcn_readlane((int)to, 63) + upto - own;
#pragma unroll
        for (int j = 0; j < E::kVec; ++j) {
          if (in[j] && to < room) list[to] = composite(key_of(v[j]), (uint32_t)(at + j));
          to += in[j] ? 1u : 0u;
        }
      }
    }
    __syncthreads();
    if (t == 0) a.gathered[(int64_t)row * kSharesMax + share] = gathered;
  });
}

// The exact cuts of a request's rows that need it, by as many workgroups as there are rows, up to kSettleRows; the last of
// them decides. 13 us for top_p alone (about 300 entries in the window: a round among cells, then ranks), 17 where top_k
// 1,000 comes first; two workgroups at most took 25, for the requests with four such rows.
template <int DT>
__global__ __launch_bounds__(kSettleThreads) void verify_settle_kernel(VerifyArgs a) {
  using E = Elem<DT>;
  __shared__ SettleScratch s;
  const int request = (int)blockIdx.x, t = (int)threadIdx.x;
  const Needed needed = a.needed[request];
  const Setting set = setting_of(a, request);
  const Place place = place_of(a, request);  // (three loads on their way together)
  const int workgroups = min((int)(__popcll(needed.slots[0]) + __popcll(needed.slots[1])), kSettleRows);
  if ((int)blockIdx.y >= workgroups) return;
  each_needed(needed, (int)blockIdx.y, kSettleRows, [&](int slot) {
    const int row = request * a.slots + slot;
    RowDist d = a.dists[row];
    const RowCut window = a.cuts[row];
    const SlotRow source = row_of<DT>(a, place, set.kind, slot);
    Candidates<DT> left(source.base, a.vocab, window, s);
    if (a.bins) left.take(a.bins + (int64_t)row * a.parts * kBins, a.gathered + (int64_t)row * kSharesMax, a.shares, share_room(a));
    if (!left.resident) left.fill();
    settle_row<DT>(a, set, window, left, d, s);
    if (t == 0) {
      if (source.drafted >= 0) {
        const int token = a.drafts[source.drafted];
        const float x = token >= 0 && token < a.vocab ? E::widen(((const typename E::Bits *)source.base)[token]) : -INFINITY;
        d.drafted = share_of(d, set, token, a.vocab, x);
      }
      a.dists[row] = d;
    }
  });
  if (workgroups > 1) {
    if (t == 0) s.last = __hip_atomic_fetch_add(&a.needed[request].settled, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)workgroups - 1;
    __syncthreads();
    if (!s.last) return;
  }
  __syncthreads();
  for (int slot = t; slot < a.slots; slot += kSettleThreads) s.dists[slot] = a.dists[request * a.slots + slot];
  __syncthreads();
  const Verdict verdict = verdict_of(a, request, set, place, s.dists, s.shared);
  if (t == 0) a.decisions[request] = decision_of(a, request, set, place, s.dists, verdict);
}

// What a thread's elements of a segment weigh in a request's draw: `rest` of them is drawn from, or `all` where nothing rests.
template <int DT>
struct RestOf {
  using E = Elem<DT>;
  using Bits = typename E::Bits;
  static constexpr int kThreads = kSegment / E::kVec;  // 16 bytes to a thread
  double rest[E::kVec], all[E::kVec];
  static __device__ __forceinline__ double share(uint64_t threshold, float max, double inverse, double scale, float x, int e) {
    if (!(x > -INFINITY) || composite(key_of(x), (uint32_t)e) < threshold) return 0.0;
    // Below e^-690 there is nothing: what is left of a P that is Q, or comes first at a uniform of zero, must not be that.
    const double d = ((double)x - (double)max) * inverse;
    return d >= -690.0 ? exp_64(d) * scale : 0.0;
  }
  __device__ __forceinline__ RestOf(const VerifyArgs &a, const Decision &d, int first) {
    const int vocab = a.vocab;
    const bool both = d.draw == kFromRest;
    const u32x4 none = {0, 0, 0, 0};
    const u32x4 p = first < vocab ? load_values<DT, false>((const Bits *)a.logits + d.target, first, vocab) : none;
    const u32x4 q = both && first < vocab ? load_values<DT, false>((const Bits *)a.draft_logits + d.draft, first, vocab) : none;
    float x[E::kVec], y[E::kVec];
    E::widen16(p, x);
    E::widen16(q, y);
#pragma unroll
    for (int j = 0; j < E::kVec; ++j) {
      const int e = first + j;
      const bool in = e < vocab;
      all[j] = in ? share(d.threshold, d.max, d.inverse, d.of_target, x[j], e) : 0.0;
      rest[j] = e == d.token ? 0.0 : all[j];
      if (both) rest[j] = fmax(all[j] - (in ? share(d.draft_threshold, d.draft_max, d.inverse, d.of_draft, y[j], e) : 0.0), 0.0);
    }
  }
};

template <int DT>
__global__ __launch_bounds__(RestOf<DT>::kThreads) void verify_weigh_kernel(VerifyArgs a) {
  constexpr int kWavesN = RestOf<DT>::kThreads / 64;
  __shared__ double wave_space[2][kWavesN];
  const int request = (int)blockIdx.y, segment = (int)blockIdx.x, t = (int)threadIdx.x;
  const Decision d = a.decisions[request];
  if (d.draw == kDone) return;
  const RestOf<DT> own(a, d, segment * kSegment + t * RestOf<DT>::E::kVec);
  double left = 0.0, all = 0.0;
#pragma unroll
  for (int j = 0; j < RestOf<DT>::E::kVec; ++j) {
    left += own.rest[j];
    all += own.all[j];
  }
  left = wave_sum(left);
  all = wave_sum(all);
  if ((t & 63) == 0) {
    wave_space[0][t >> 6] = left;
    wave_space[1][t >> 6] = all;
  }
  __syncthreads();
  if (t >= 64) return;
  left = wave_sum(t < kWavesN ? wave_space[0][t] : 0.0);
  all = wave_sum(t < kWavesN ? wave_space[1][t] : 0.0);
  if (t == 0) a.segment_sums[(int64_t)request * a.segments + segment] = double2{left, all};
}

template <int DT>
__global__ __launch_bounds__(RestOf<DT>::kThreads) void verify_pick_kernel(VerifyArgs a) {
  constexpr int kThreads = RestOf<DT>::kThreads, kWavesN = kThreads / 64;
  __shared__ double wave_space[kWavesN], befores[kWavesN];
  __shared__ int places[kWavesN], tokens[kWavesN];
  __shared__ bool reaches[kWavesN];
  const int request = (int)blockIdx.x, t = (int)threadIdx.x;
  const Decision d = a.decisions[request];
  if (d.draw == kDone) return;
  const double2 *sums = a.segment_sums + (int64_t)request * a.segments;
  // A run of segments to a thread.
  const int per = (a.segments + kThreads - 1) / kThreads, begin = min(t * per, a.segments), end = min(begin + per, a.segments);
  double own = 0.0, own_all = 0.0, total;
  for (int i = begin; i < end; ++i) {
    own += sums[i].x;
    own_all += sums[i].y;
  }
  double before = block_prefix<kWavesN>(own, wave_space, total) - own;
  const bool plain = !(total > 0.0);  // nothing left: P is Q, but for roundings
  if (plain) before = block_prefix<kWavesN>(own_all, wave_space, total) - own_all;
  const double goal = d.uniform * total;
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
  // Of a wave: its first lane that has one, or its last with a weight. Then of the waves. (Atomics on one word go lane by
  // lane: 2 us here and 4 below.)
  auto settle_on = [&](bool reach, bool some) {
    const uint64_t reached = __ballot(reach), weighted = __ballot(some);
    return reached ? (int)__builtin_ctzll(reached) : weighted ? 63 - (int)__builtin_clzll(weighted) : -1;
  };
  auto first_wave = [&]() {
    int wave = -1;
    bool sure = false;
#pragma unroll
    for (int w = 0; w < kWavesN; ++w) {
      if (!sure && places[w] >= 0) {
        wave = w;
        sure = reaches[w];
      }
    }
    return wave;
  };
  const int wave = t >> 6, lane = t & 63;
  const bool reach = found < a.segments;
  const int owner = settle_on(reach, last >= 0);
  if (lane == max(owner, 0)) {
    places[wave] = owner < 0 ? -1 : reach ? found : last;
    befores[wave] = reach ? found_before : last_before;
    reaches[wave] = reach;
  }
  __syncthreads();
  const int of = first_wave(), chosen = of < 0 ? 0 : places[of];
  const double chosen_before = of < 0 ? 0.0 : befores[of];
  const int first = chosen * kSegment + t * RestOf<DT>::E::kVec;
  const RestOf<DT> weights(a, d, first);
  double sum = 0.0, all;
#pragma unroll
  for (int j = 0; j < RestOf<DT>::E::kVec; ++j) sum += plain ? weights.all[j] : weights.rest[j];
  double run = block_prefix<kWavesN>(sum, wave_space, all) - sum + chosen_before;
  int token = a.vocab, some = -1;
#pragma unroll
  for (int j = 0; j < RestOf<DT>::E::kVec; ++j) {
    const double w = plain ? weights.all[j] : weights.rest[j];
    run += w;
    if (w > 0.0) {
      some = first + j;
      if (token == a.vocab && run > goal) token = first + j;
    }
  }
  const bool in = token < a.vocab;
  const int holder = settle_on(in, some >= 0);
  if (lane == max(holder, 0)) {
    places[wave] = holder;
    reaches[wave] = in;
    tokens[wave] = in ? token : some;
  }
  __syncthreads();
  if (t == 0) {
    const int w = first_wave();
    a.tokens[d.out] = w < 0 ? 0 : tokens[w];
  }
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

constexpr int kPartMin = 16384;  // half as much makes twice the lists to bring together: one request of four tokens, 23.6 us against 22.8

// Rows are cut into parts, a workgroup each, until there are some to a compute unit.
int verify_parts(int64_t rows, int vocab) {
  const int64_t parts = std::min<int64_t>({kBlocksAimed / std::max<int64_t>(rows, 1), (vocab + kPartMin - 1) / kPartMin, kPartsMax});
  return (int)std::max<int64_t>(parts, 1);
}

// Lists (parts of rows) that there may be: rows that are cut make at most kBlocksAimed of them.
int64_t lists_max(int64_t rows) { return std::max<int64_t>(rows, kBlocksAimed); }

int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// The workspace's arrays: where each begins, and the end.
struct Space { int64_t sums, entries, dists, bins, groups, pools, decisions, cuts, needed, gathered, segments, end; };
constexpr int64_t kBinnedMax = 4096;  // lists (parts of rows) that have bins, 16 KB each
Space space_of(int64_t requests, int64_t slots, int64_t lists, int64_t segments) {
  Space s;
  s.sums = 0;
  s.entries = s.sums + aligned(lists * (int64_t)sizeof(PartSum));
  s.dists = s.entries + aligned(lists * kPoolMax * 8);
  s.bins = s.dists + aligned(requests * slots * (int64_t)sizeof(RowDist));
  s.groups = s.bins + std::min(lists, kBinnedMax) * kBins * 8;
  s.pools = s.groups + std::min(lists, kBinnedMax) * kGroups * (int64_t)sizeof(double2);
  s.decisions = s.pools + aligned(requests * slots * kPoolMax * 8);
  s.cuts = s.decisions + aligned(requests * (int64_t)sizeof(Decision));
  s.needed = s.cuts + aligned(requests * slots * (int64_t)sizeof(RowCut));
  s.gathered = s.needed + aligned(requests * (int64_t)sizeof(Needed));
  s.segments = s.gathered + aligned(requests * slots * kSharesMax * 4);
  s.end = s.segments + aligned(requests * segments * (int64_t)sizeof(double2));
  return s;
}

template <int DT>
int launch_verify(const VerifyArgs &a, hipStream_t s) {
  const unsigned rows = (unsigned)(a.requests * a.slots), blocks = rows * (unsigned)a.parts;
  // Four or eight waves where they have a chunk each. Else, up to a workgroup for each compute unit, sixteen.
  if (a.part_len <= 4 * kChunk) hipLaunchKernelGGL((verify_rows_kernel<DT, 4>), dim3(blocks), dim3(256), 0, s, a);
  else if (blocks <= 256u && a.part_len > 8 * kChunk) hipLaunchKernelGGL((verify_rows_kernel<DT, 16>), dim3(blocks), dim3(1024), 0, s, a);
  else hipLaunchKernelGGL((verify_rows_kernel<DT, 8>), dim3(blocks), dim3(512), 0, s, a);
  TABBY_HIP_CHECK(hipGetLastError());
  auto decide = [&](auto full) {
    constexpr bool kFull = decltype(full)::value;
    if (a.slots <= 4) hipLaunchKernelGGL((verify_decide_kernel<DT, 4, kFull>), dim3((unsigned)a.requests), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((verify_decide_kernel<DT, 16, kFull>), dim3((unsigned)a.requests), dim3(1024), 0, s, a);
    return hipGetLastError();
  };
  if (a.whole) TABBY_HIP_CHECK(decide(std::true_type{}));
  else TABBY_HIP_CHECK(decide(std::false_type{}));
  if (!a.whole) return TABBY_OK;
  if (a.bins) {
    hipLaunchKernelGGL(verify_gather_kernel<DT>, dim3((unsigned)a.shares, (unsigned)a.requests, kGatherRows), dim3(kGatherThreads), 0, s, a);
    TABBY_HIP_CHECK(hipGetLastError());
  }
  hipLaunchKernelGGL(verify_settle_kernel<DT>, dim3((unsigned)a.requests, kSettleRows), dim3(kSettleThreads), 0, s, a);
  TABBY_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL(verify_weigh_kernel<DT>, dim3((unsigned)a.segments, (unsigned)a.requests), dim3(RestOf<DT>::kThreads), 0, s, a);
  TABBY_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL(verify_pick_kernel<DT>, dim3((unsigned)a.requests), dim3(RestOf<DT>::kThreads), 0, s, a);
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
  // For these sizes and every smaller one.
  const int64_t slots = 2 * drafts_max + 1;
  *bytes = space_of(requests, slots, lists_max(requests * slots), ((int64_t)vocab + kSegment - 1) / kSegment).end;
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
  const int fit = (int)std::max<int64_t>(1, std::min<int64_t>(parts, lists_max((int64_t)requests * slots) / ((int64_t)requests * slots)));
  const int part_len = (int)((((int64_t)vocab + fit - 1) / fit + 31) / 32 * 32);
  const int used = (int)(((int64_t)vocab + part_len - 1) / part_len);
  const int segments = (vocab + kSegment - 1) / kSegment;
  const int64_t lists = (int64_t)requests * slots * used;
  // As many workgroups as the chip holds at once, with some loads each.
  const int shares = std::max(std::min({kGatherBlocks / requests, vocab / 4096, kSharesMax}), 1);
  const Space space = space_of(requests, slots, lists, segments);
  char *w = (char *)workspace_dev;
  VerifyArgs a{logits_dev, draft_logits_dev, row_stride, draft_row_stride, drafts_dev, uniforms_dev, offsets_dev, params_dev,
               rows, requests, drafts_max, vocab, slots, (flags & TABBY_FLAG_FULL_VOCAB) != 0, used, part_len, segments,
               tokens_dev, accepted_dev, status_dev, (PartSum *)(w + space.sums), (uint64_t *)(w + space.entries),
               (RowDist *)(w + space.dists), lists <= kBinnedMax ? (uint64_t *)(w + space.bins) : nullptr,
               (uint64_t *)(w + space.pools), (Decision *)(w + space.decisions), (double2 *)(w + space.segments),
               (RowCut *)(w + space.cuts), (Needed *)(w + space.needed), (double2 *)(w + space.groups), (uint32_t *)(w + space.gathered), shares};
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
