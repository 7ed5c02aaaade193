// Which memory a call writes beside what it reads: the check that turns down outputs over inputs that are still read.
// Blocks of a grid read and write in no order, so an overlap that is no update in place would give results that depend
// on timing.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <numeric>

namespace ogx {

// A call's memory as runs of `width` bytes, one for every point of up to three axes.  Strides in bytes.
struct Region {
  const char* base;
  int64_t width, n[3], stride[3];
};

inline Region rows_region(const void* base, int64_t size, int64_t width, int64_t batch, int64_t stride_b,
                          int64_t tokens, int64_t stride_t) {
  return Region{static_cast<const char*>(base), base == nullptr ? 0 : width * size, {1, batch, tokens},
                {0, stride_b * size, stride_t * size}};
}
inline Region flat_region(const void* base, int64_t bytes) { return rows_region(base, 1, bytes, 1, 0, 1, 0); }

using Wide = __int128;  // a stride of 2^39 bytes times 2^25 tokens is past 64 bits

// The bytes from a region's base that its axes from `axis` on reach: [low, high).
inline void region_extent(const Region& r, int axis, Wide* low, Wide* high) {
  *low = 0;
  *high = r.width;
  for (int i = axis; i < 3; ++i) (r.stride[i] < 0 ? *low : *high) += static_cast<Wide>(r.n[i] - 1) * r.stride[i];
}

// Whether a byte of `b`, whose base lies `apart` bytes behind `a`'s, can be one of `a`'s; the axes before `axis` are left
// out.  False is certain.  True is, too, but for regions that lie in one another with unlike strides, which are called
// overlapping.
inline bool regions_meet(const Region& a, const Region& b, Wide apart, int axis) {
  Wide a_low, a_high, b_low, b_high;
  region_extent(a, axis, &a_low, &a_high);
  region_extent(b, axis, &b_low, &b_high);
  if (apart + b_low >= a_high || apart + b_high <= a_low) return false;
  // columns of the same rows: all runs start at multiples of one step from their base
  int64_t step = 0;
  for (int i = axis; i < 3; ++i) {
    if (a.n[i] > 1) step = std::gcd(step, a.stride[i]);
    if (b.n[i] > 1) step = std::gcd(step, b.stride[i]);
  }
  if (step > 0) {
    const Wide at = (apart % step + step) % step;
    if (at >= a.width && at + b.width <= step) return false;
  }
  if (axis == 3) return true;
  // the outermost axis is left out where it moves neither, or both by more than the others reach: then only a
  // neighbour on either side can meet
  const int64_t move = a.n[axis] > 1 ? a.stride[axis] : b.stride[axis];
  if (a.n[axis] == 1 && b.n[axis] == 1) return regions_meet(a, b, apart, axis + 1);
  if (a.n[axis] > 1 && b.n[axis] > 1 && a.stride[axis] != b.stride[axis]) return true;
  region_extent(a, axis + 1, &a_low, &a_high);
  region_extent(b, axis + 1, &b_low, &b_high);
  if (move <= 0 || a_low < 0 || b_low < 0 || a_high > move || b_high > move) return true;
  const Wide at = (apart % move + move) % move;
  return regions_meet(a, b, at, axis + 1) || regions_meet(a, b, at - move, axis + 1);
}

inline bool meet(const Region& a, const Region& b) {
  return a.width > 0 && b.width > 0 && regions_meet(a, b, static_cast<Wide>(b.base - a.base), 0);
}

// The same bytes in the same order: an update in place.
inline bool same_region(const Region& a, const Region& b) {
  if (a.base != b.base || a.width != b.width) return false;
  for (int i = 0; i < 3; ++i)
    if (a.n[i] != b.n[i] || (a.n[i] > 1 && a.stride[i] != b.stride[i])) return false;
  return true;
}

// Whether the runs of an output are apart from one another: tokens, and batches behind or between them.
inline bool runs_apart(const Region& r) {
  const auto size = [](Wide v) { return v < 0 ? -v : v; };
  const Wide batch = r.n[1], tokens = r.n[2], sb = size(r.stride[1]), st = size(r.stride[2]);
  if (tokens > 1 && st < r.width) return false;
  return batch == 1 || sb >= (tokens - 1) * st + r.width ||
         (sb >= r.width && (tokens == 1 || st >= (batch - 1) * sb + r.width));
}

// An output may meet neither another output nor an input, but those it may be an update of.
struct Output {
  Region at;
  int in_place[2];  // inputs, or -1
};

template <size_t O, size_t I>
bool outputs_ok(const Output (&outputs)[O], const Region (&inputs)[I]) {
  Wide low[O + I], high[O + I];  // addresses: most regions are apart by these alone
  for (size_t i = 0; i < O + I; ++i) {
    const Region& r = i < O ? outputs[i].at : inputs[i - O];
    region_extent(r, 0, &low[i], &high[i]);
    low[i] += reinterpret_cast<intptr_t>(r.base);
    high[i] += reinterpret_cast<intptr_t>(r.base);
  }
  for (size_t o = 0; o < O; ++o) {
    const Region& at = outputs[o].at;
    if (at.width > 0 && !runs_apart(at)) return false;
    for (size_t i = o + 1; i < O + I; ++i) {
      if (low[i] >= high[o] || low[o] >= high[i]) continue;
      if (i < O) {
        if (meet(at, outputs[i].at)) return false;
        continue;
      }
      const int input = static_cast<int>(i - O);
      const bool update = outputs[o].in_place[0] == input || outputs[o].in_place[1] == input;
      if (!(update && same_region(at, inputs[input])) && meet(at, inputs[input])) return false;
    }
  }
  return true;
}

}  // namespace ogx
