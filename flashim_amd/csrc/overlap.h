// Whether strided tensors share memory, exactly: plain C++, built for the torch operators and for the CPU tests.
//
// Elements of two tensors meet where sum_k s_k v_k, v_k from ranges that their sizes give (a dimension of either; one range where both
// step alike), comes within an element's width of the distance between them. Dimensions are taken by falling stride, each with the
// values that the smaller ones can still make up for: two or three where strides nest, as views of one buffer do.
#pragma once

#include <stdint.h>

#include <algorithm>
#include <vector>

namespace fim {

struct Strided {
  int64_t at = 0;   // first byte
  int64_t es = 1;   // bytes of an element, or of neighbours
  struct Dim {
    int64_t stride, size;  // bytes, elements
  };
  std::vector<Dim> dims;  // of two elements or more
  int64_t end() const {
    int64_t e = at + es;
    for (const Dim& d : dims) e += d.stride * (d.size - 1);
    return e;
  }
};

class Meeting {
 public:
  // Past this many partial sums, strides that do not nest count as ones that meet
  static constexpr int MOST = 1 << 16;

  static bool of(const Strided& a, const Strided& b) {
    Meeting m;
    for (const auto& d : a.dims) m.add(d.stride, 0, d.size - 1);
    for (const auto& d : b.dims) m.add(d.stride, 1 - d.size, 0);
    if (m.axes.empty()) return a.at < b.at + b.es && b.at < a.at + a.es;
    m.order();
    const int64_t apart = b.at - a.at;
    return m.reaches(0, apart - (a.es - 1), apart + (b.es - 1));
  }
  // Whether two elements of one tensor meet: a difference of their indices, its first value that is not 0 above it
  static bool of(const Strided& a) {
    if (a.dims.empty() || (a.dims.size() == 1 && a.dims[0].stride >= a.es)) return false;
    Meeting m;
    for (const auto& d : a.dims) m.axes.push_back({d.stride, 1 - d.size, d.size - 1});
    m.order();
    for (size_t k = 0; k < m.axes.size(); ++k) {
      const Axis whole = m.axes[k];
      m.axes[k].from = 1;
      m.rest();
      if (m.reaches(k, 1 - a.es, a.es - 1)) return true;
      m.axes[k] = whole;
    }
    return false;
  }

 private:
  struct Axis {
    int64_t stride, from, to;
  };
  std::vector<Axis> axes;
  std::vector<int64_t> least, most;  // of the sums from an axis on
  int left = MOST;

  void add(int64_t stride, int64_t from, int64_t to) {
    for (Axis& x : axes)
      if (x.stride == stride) {
        x.from += from;
        x.to += to;
        return;
      }
    axes.push_back({stride, from, to});
  }
  void order() {
    std::sort(axes.begin(), axes.end(), [](const Axis& a, const Axis& b) { return a.stride > b.stride; });
    rest();
  }
  void rest() {
    least.assign(axes.size() + 1, 0);
    most.assign(axes.size() + 1, 0);
    for (size_t k = axes.size(); k-- > 0;) {
      least[k] = least[k + 1] + axes[k].stride * axes[k].from;
      most[k] = most[k + 1] + axes[k].stride * axes[k].to;
    }
  }
  static int64_t floor_div(int64_t n, int64_t d) { return n / d - (n % d < 0); }

  // Whether the axes from k on have a sum in [lo, hi]
  bool reaches(size_t k, int64_t lo, int64_t hi) {
    if (hi < least[k] || lo > most[k]) return false;
    if (k == axes.size()) return true;  // (0 is in it)
    if (--left < 0) return true;
    const Axis& x = axes[k];
    if (x.stride == 0) return reaches(k + 1, lo, hi);
    int64_t from = -floor_div(most[k + 1] - lo, x.stride), to = floor_div(hi - least[k + 1], x.stride);
    from = std::max(from, x.from);
    to = std::min(to, x.to);
    for (int64_t v = from; v <= to; ++v)
      if (reaches(k + 1, lo - x.stride * v, hi - x.stride * v)) return true;
    return false;
  }
};

// Tensors of a call, of which none that is written may meet another, or itself
class Extents {
 public:
  void add(const Strided& t, bool written) { all.push_back({t, t.end(), written}); }
  bool apart() {
    std::sort(all.begin(), all.end(), [](const One& a, const One& b) { return a.t.at < b.t.at; });
    std::vector<const One*> open;  // those whose ends are not behind yet
    for (const One& e : all) {
      if (e.written && Meeting::of(e.t)) return false;
      size_t kept = 0;
      for (const One* o : open)
        if (o->end > e.t.at) open[kept++] = o;
      open.resize(kept);
      for (const One* o : open)
        if ((e.written || o->written) && Meeting::of(o->t, e.t)) return false;
      open.push_back(&e);
    }
    return true;
  }

 private:
  struct One {
    Strided t;
    int64_t end;
    bool written;
  };
  std::vector<One> all;
};

}  // namespace fim
