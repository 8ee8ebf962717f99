// Which memory an entry point's operands take, from their addresses, extents and strides, and whether an output
// shares any of it: host arithmetic of some 10 ns a pair, where tensors cost the caller 3 us.
#pragma once

#include <stdint.h>

#include <algorithm>
#include <initializer_list>

namespace kf {

struct Axis {
  int64_t n, stride;  // elements
};

// The elements of one operand; null or without elements: no memory.
struct Region {
  static constexpr int MOST = 4;
  using Wide = __int128;  // extents times strides of any size
  const char* name = "";
  const void* at = nullptr;
  int elem = 0;  // bytes
  int dims = 0;
  Axis axes[MOST];

  Region(const char* what, const void* where, int bytes, std::initializer_list<Axis> all) : name(what), at(where), elem(bytes) {
    for (const Axis& a : all) {
      if (a.n <= 0) at = nullptr;
      axes[dims++] = a;
    }
  }
  Wide first() const { return static_cast<Wide>(reinterpret_cast<uintptr_t>(at)); }
  Wide past() const {
    Wide span = 1;
    for (int i = 0; i < dims; ++i) span += static_cast<Wide>(axes[i].n - 1) * axes[i].stride;
    return first() + span * elem;
  }
  // Whether two of its indexes may name one element: false only where each stride passes all that the shorter ones span.
  bool overlaps_itself() const {
    if (at == nullptr) return false;
    Axis up[MOST];
    std::copy(axes, axes + dims, up);
    std::sort(up, up + dims, [](const Axis& a, const Axis& b) { return a.stride < b.stride; });
    Wide span = 0;
    for (int i = 0; i < dims; ++i) {
      if (up[i].n == 1) continue;
      if (up[i].stride <= span) return true;
      span += static_cast<Wide>(up[i].n - 1) * up[i].stride;
    }
    return false;
  }
  bool same_place(const Region& o) const {
    if (at != o.at || elem != o.elem || dims != o.dims) return false;
    for (int i = 0; i < dims; ++i)
      if (axes[i].n != o.axes[i].n || (axes[i].n > 1 && axes[i].stride != o.axes[i].stride)) return false;
    return true;
  }
};

// An axis that two operands have in common: their extents along it.
struct CommonAxis {
  int64_t stride, a, b;
};

// Whether delta is a sum of i * stride over the axes, longest stride first, with -b < i < a on each.
inline bool regions_meet(const CommonAxis* axis, int left, Region::Wide delta) {
  using Wide = Region::Wide;
  if (left == 0) return delta == 0;
  if (axis->a == 1 && axis->b == 1) return regions_meet(axis + 1, left - 1, delta);
  const Wide stride = axis->stride;
  if (stride <= 0) return true;
  Wide low = 0, high = 0;
  for (int i = 1; i < left; ++i) {
    low -= static_cast<Wide>(axis[i].b - 1) * axis[i].stride;
    high += static_cast<Wide>(axis[i].a - 1) * axis[i].stride;
  }
  const auto down = [](Wide x, Wide by) { return x >= 0 ? x / by : -((-x + by - 1) / by); };
  const Wide from = std::max<Wide>(1 - axis->b, -down(high - delta, stride));
  const Wide to = std::min<Wide>(axis->a - 1, down(delta - low, stride));
  if (to - from > 64) return true;
  for (Wide i = from; i <= to; ++i)
    if (regions_meet(axis + 1, left - 1, delta - i * stride)) return true;
  return false;
}

// Whether they share memory: exact for operands of one type and of equal strides (parts of one buffer), and true for
// others whose addresses meet.
inline bool overlap(const Region& a, const Region& b) {
  if (a.at == nullptr || b.at == nullptr || b.first() >= a.past() || a.first() >= b.past()) return false;
  const Region::Wide delta = b.first() - a.first();
  if (a.elem != b.elem || a.dims != b.dims || delta % a.elem != 0) return true;
  CommonAxis axes[Region::MOST];
  for (int i = 0; i < a.dims; ++i) {
    const Axis &x = a.axes[i], &y = b.axes[i];
    if (x.n > 1 && y.n > 1 && x.stride != y.stride) return true;
    axes[i] = {x.n > 1 ? x.stride : y.stride, x.n, y.n};
  }
  std::sort(axes, axes + a.dims, [](const CommonAxis& x, const CommonAxis& y) { return x.stride > y.stride; });
  return regions_meet(axes, a.dims, delta / a.elem);
}

}  // namespace kf
