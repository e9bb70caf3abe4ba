// Beam search's states follow the beams that survived: row (g, b) of every state becomes what row
// (g, parent[g, b]) was, in the first len_g positions of each of its segments, for many states in one
// launch, in place or into a second set of buffers.
//
// One lane owns one column -- BYTES consecutive bytes at one place of the group's rows -- and holds it for
// all of the group's beams: it loads the columns of the parents, then stores them. So a lane never
// reads what another writes and the move may run in place, whatever the parents; and a parent with
// several children is fetched from memory once, its further reads close behind in the cache. Bound by
// HBM: every surviving row read once, every moved row written once. Stores bypass the caches, which leaves
// these to the parents' further reads: 48 states of [64, 2, 1024, 64] bf16, 16 groups of different lengths,
// 136 to 142 us, one card or another (5.0 to 5.2 TB/s; through the caches 146); 12 beams of 24 states of
// [48, 2, 1024, 128], 98 us (6.7 TB/s; 130).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <memory>
#include <new>
#include <string>

#include "abi_internal.h"
#include "loads.h"

namespace tabby {
namespace {

constexpr int kReorderBlock = 256;
constexpr int kReorderBeams = 64;
constexpr int kStatesPerLaunch = 64;  // their addresses travel as arguments

struct ReorderArgs {
  const char *src[kStatesPerLaunch];
  char *dst[kStatesPerLaunch];
  int beams, segments;
  int64_t capacity;  // positions of a segment
  int64_t unit;      // bytes of a position
  int64_t row_stride, segment_stride;
  const int32_t *parents, *lengths;
  uint32_t chunks;  // columns' workgroups to a segment
  uint32_t first;   // of all groups' segments' workgroups, this launch's first
};
constexpr int64_t kReorderGrid = 1 << 23;  // of 256 threads: 2^32 in a launch are too many

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
template <int BYTES>
struct ColumnOf;
template <>
struct ColumnOf<16> { using T = u32x4; };
template <>
struct ColumnOf<8> { using T = u32x2_t; };
template <>
struct ColumnOf<4> { using T = uint32_t; };
template <>
struct ColumnOf<2> { using T = uint16_t; };
template <>
struct ColumnOf<1> { using T = uint8_t; };

// NB: beams held at once. Grid: ((group * segments + segment) * chunks + chunk - first, state).
template <int BYTES, int NB, bool IN_PLACE>
__global__ __launch_bounds__(kReorderBlock, 4) void beam_reorder_kernel(ReorderArgs a) {
  using T = typename ColumnOf<BYTES>::T;
  const uint32_t id = a.first + blockIdx.x;
  const uint32_t line = id / a.chunks, chunk = id - line * a.chunks;
  const int g = (int)(line / (uint32_t)a.segments), seg = (int)(line - (uint32_t)g * a.segments);
  int64_t length = a.capacity;
  if (a.lengths) length = min(length, (int64_t)max(a.lengths[g], 0));
  const int64_t at = ((int64_t)chunk * kReorderBlock + threadIdx.x) * BYTES;
  if (at >= length * a.unit) return;
  const int64_t first = (int64_t)g * a.beams * a.row_stride + seg * a.segment_stride + at;
  const char *src = a.src[blockIdx.y] + first;
  char *dst = a.dst[blockIdx.y] + first;
  const int32_t *parents = a.parents + (int64_t)g * a.beams;
  uint32_t parent[NB];
  T v[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    parent[b] = b < a.beams ? (uint32_t)__builtin_amdgcn_readfirstlane(parents[b]) : ~0u;
    if (IN_PLACE && parent[b] == (uint32_t)b) parent[b] = ~0u;
  }
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (parent[b] < (uint32_t)a.beams) v[b] = *reinterpret_cast<const T *>(src + parent[b] * a.row_stride);
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (parent[b] < (uint32_t)a.beams) __builtin_nontemporal_store(v[b], reinterpret_cast<T *>(dst + b * a.row_stride));
}

template <int BYTES, int NB>
int launch_width(ReorderArgs &a, int groups, int states, bool in_place, hipStream_t s) {
  const int64_t chunks = (a.capacity * a.unit + (int64_t)kReorderBlock * BYTES - 1) / ((int64_t)kReorderBlock * BYTES);
  const int64_t rows = (int64_t)groups * a.segments;
  if (chunks > INT32_MAX / rows) return record_failure(TABBY_EINVAL, "the states are too large for one call");
  a.chunks = (uint32_t)chunks;
  for (int64_t first = 0; first < chunks * rows; first += kReorderGrid) {
    a.first = (uint32_t)first;
    const dim3 grid((unsigned)std::min(chunks * rows - first, kReorderGrid), (unsigned)states);
    if (in_place) hipLaunchKernelGGL((beam_reorder_kernel<BYTES, NB, true>), grid, dim3(kReorderBlock), 0, s, a);
    else hipLaunchKernelGGL((beam_reorder_kernel<BYTES, NB, false>), grid, dim3(kReorderBlock), 0, s, a);
    TABBY_HIP_CHECK(hipGetLastError());
  }
  return TABBY_OK;
}

// Columns of at most 256 bytes / beams: a lane holds one for each beam, 64 registers of them.
template <int BYTES>
int launch_reorder(ReorderArgs &a, int groups, int states, bool in_place, hipStream_t s) {
  if (a.beams <= 4) return launch_width<BYTES, 4>(a, groups, states, in_place, s);
  if (a.beams <= 8) return launch_width<BYTES, 8>(a, groups, states, in_place, s);
  if (a.beams <= 16) return launch_width<BYTES, 16>(a, groups, states, in_place, s);
  if (a.beams <= 32) return launch_width<(BYTES < 8 ? BYTES : 8), 32>(a, groups, states, in_place, s);
  return launch_width<(BYTES < 4 ? BYTES : 4), 64>(a, groups, states, in_place, s);
}

// What one state takes of memory.
struct StateShape {
  int64_t rows, row_stride;
  int64_t segments, segment_stride, segment;
  int64_t extent() const { return (segments - 1) * segment_stride + segment; }  // of a row
  int64_t span() const { return (rows - 1) * row_stride + extent(); }
};

// Whether a state and one `apart` bytes after it share any byte; apart < span. Rows do not interleave, and segments
// do not, so that of either only the two nearest can meet.
bool states_meet(const StateShape &s, int64_t apart) {
  const int64_t row = s.rows > 1 ? apart / s.row_stride : 0;
  for (int64_t r = row; r < std::min(row + 2, s.rows); ++r) {
    const int64_t rest = std::abs(apart - r * s.row_stride);
    const int64_t segment = s.segments > 1 ? rest / s.segment_stride : 0;
    for (int64_t i = segment; i < std::min(segment + 2, s.segments); ++i)
      if (std::abs(rest - i * s.segment_stride) < s.segment) return true;
  }
  return false;
}

struct StateAt {
  int64_t address;
  bool read_only;  // two of these may share memory
};

// Whether any two states share memory that one of them has written to. Sorts them.
bool any_meet(StateAt *at, size_t n, const StateShape &s) {
  const auto before = [](const StateAt &a, const StateAt &b) { return a.address < b.address; };
  if (!std::is_sorted(at, at + n, before)) std::sort(at, at + n, before);
  // Nearly always states lie one after another, or side by side within a row's stride (layers in one tensor).
  const int64_t extent = s.extent(), span = s.span();
  size_t first = 0, i = 1;  // `first`: of those side by side
  for (; i < n; ++i) {
    const int64_t from_first = at[i].address - at[first].address;
    if (first + 1 == i ? from_first >= span : from_first / s.row_stride >= s.rows) first = i;
    else if (s.rows < 2 || at[i].address - at[i - 1].address < extent || from_first + extent > s.row_stride) break;
  }
  if (i >= n) return false;
  for (i = 0; i < n; ++i)
    for (size_t j = i + 1; j < n && at[j].address - at[i].address < span; ++j)
      if (!(at[i].read_only && at[j].read_only) && states_meet(s, at[j].address - at[i].address)) return true;
  return false;
}

int check_states_apart(const void *const *src, void *const *dst, int states, bool in_place, const StateShape &s) {
  const size_t n = (size_t)states * (in_place ? 1 : 2);
  StateAt few[256];
  std::unique_ptr<StateAt[]> many;
  if (n > sizeof(few) / sizeof(few[0])) {
    many.reset(new (std::nothrow) StateAt[n]);
    if (!many) return record_failure(TABBY_EINVAL, "no memory to look at that many states");
  }
  StateAt *at = many ? many.get() : few;
  for (int i = 0; i < states; ++i) {
    at[i] = {(int64_t)(uintptr_t)dst[i], false};
    if (!in_place) at[states + i] = {(int64_t)(uintptr_t)src[i], true};
  }
  if (any_meet(at, n, s))
    return record_failure(TABBY_EINVAL, in_place ? "states moved in place must not overlap each other"
                                                 : "destinations must not overlap sources or each other");
  return TABBY_OK;
}

}  // namespace
}  // namespace tabby

using namespace tabby;

extern "C" int tabby_beam_reorder_device(const void *const *src_dev, void *const *dst_dev, int32_t states,
                                         int32_t groups, int32_t beams, int32_t segments, int64_t capacity,
                                         int64_t unit_bytes, int64_t row_stride, int64_t segment_stride,
                                         const int32_t *parents_dev, const int32_t *lengths_dev, void *stream) {
  if (!src_dev || !dst_dev || !parents_dev) return record_failure(TABBY_EINVAL, "null pointer");
  if (states < 1 || groups < 1 || segments < 1 || capacity < 1 || unit_bytes < 1)
    return record_failure(TABBY_EINVAL, "states, groups, segments, capacity and unit_bytes must be >= 1");
  if (beams < 1 || beams > kReorderBeams)
    return record_failure(TABBY_EINVAL, "beams must be between 1 and " + std::to_string(kReorderBeams) + ", got " + std::to_string(beams));
  if (capacity > INT64_MAX / unit_bytes) return record_failure(TABBY_EINVAL, "a segment must fit 63 bits");
  if (!lengths_dev) {  // whole segments: one position each, whose columns may be wide
    unit_bytes *= capacity;
    capacity = 1;
  }
  const int64_t segment = capacity * unit_bytes;
  if (segments > 1 && segment_stride < segment)
    return record_failure(TABBY_EINVAL, "segment_stride must be at least capacity x unit_bytes");
  if ((int64_t)groups * segments > INT32_MAX) return record_failure(TABBY_EINVAL, "groups x segments must fit 32 bits");
  const int64_t rows = (int64_t)groups * beams;
  const int64_t last = (segments - 1) * segment_stride;  // where a row's last segment starts
  if (rows > 1 && row_stride < last + segment) return record_failure(TABBY_EINVAL, "rows must not overlap: row_stride is too small");
  // The widest column that every address is a multiple of.
  uint64_t bits = (uint64_t)unit_bytes | (rows > 1 ? (uint64_t)row_stride : 0) | (segments > 1 ? (uint64_t)segment_stride : 0);
  const bool in_place = src_dev[0] == dst_dev[0];
  for (int i = 0; i < states; ++i) {
    const char *from = (const char *)src_dev[i], *to = (const char *)dst_dev[i];
    if (!from || !to) return record_failure(TABBY_EINVAL, "null pointer");
    if ((from == to) != in_place) return record_failure(TABBY_EINVAL, "either every state or none is moved in place");
    bits |= (uint64_t)(uintptr_t)from | (uint64_t)(uintptr_t)to;
  }
  // The move reads and writes each state on its own: what two share would be moved twice, or half.
  const int rc = check_states_apart(src_dev, dst_dev, states, in_place,
                                    {rows, rows > 1 ? row_stride : 0, segments, segments > 1 ? segment_stride : 0, segment});
  if (rc) return rc;
  const hipStream_t s = (hipStream_t)stream;
  for (int i0 = 0; i0 < states; i0 += kStatesPerLaunch) {
    const int n = std::min(kStatesPerLaunch, states - i0);
    ReorderArgs a{};
    for (int i = 0; i < n; ++i) {
      a.src[i] = (const char *)src_dev[i0 + i];
      a.dst[i] = (char *)dst_dev[i0 + i];
    }
    a.beams = beams;
    a.segments = segments;
    a.capacity = capacity;
    a.unit = unit_bytes;
    a.row_stride = row_stride;
    a.segment_stride = segment_stride;
    a.parents = parents_dev;
    a.lengths = lengths_dev;
    int rc;
    if (bits % 16 == 0) rc = launch_reorder<16>(a, groups, n, in_place, s);
    else if (bits % 8 == 0) rc = launch_reorder<8>(a, groups, n, in_place, s);
    else if (bits % 4 == 0) rc = launch_reorder<4>(a, groups, n, in_place, s);
    else if (bits % 2 == 0) rc = launch_reorder<2>(a, groups, n, in_place, s);
    else rc = launch_reorder<1>(a, groups, n, in_place, s);
    if (rc) return rc;
  }
  return TABBY_OK;
}
