// Whether two strided tensors share a byte (host).
#ifndef L20_OVERLAP_H_
#define L20_OVERLAP_H_

#include <algorithm>

#include <stdint.h>

namespace l20la {

// `width` bytes at base + i row + j head for i < rows, j < heads (strides in bytes).
struct Lattice {
  int64_t base, row, head, rows, heads, width;
  Lattice(const void *at, int64_t row_, int64_t head_, int64_t rows_, int64_t heads_, int64_t width_)
      : base((int64_t)(uintptr_t)at), row(row_), head(head_), rows(rows_), heads(heads_), width(width_) {
    flat(row, rows);
    flat(head, heads);
  }
  int64_t end() const { return base + (rows - 1) * row + (heads - 1) * head + width; }
  // Whether a piece of it meets lo .. hi - 1.
  bool meets(int64_t lo, int64_t hi) const {
    const bool by_row = row >= head;  // the longer stride first: few of its steps can reach
    const int64_t big = by_row ? row : head, bigs = by_row ? rows : heads;
    const int64_t small = by_row ? head : row, smalls = by_row ? heads : rows;
    const int64_t from = lo - width + 1 - base, to = hi - 1 - base;  // where a piece that meets it begins
    int64_t i = big ? std::max<int64_t>(0, up(from - (smalls - 1) * small, big)) : 0;
    for (; i < bigs && i * big <= to; ++i) {
      const int64_t f = from - i * big, t = to - i * big;
      if (small ? std::max<int64_t>(0, up(f, small)) <= std::min(smalls - 1, t / small) : f <= 0) return true;
      if (!big) break;
    }
    return false;
  }

 private:
  static int64_t up(int64_t a, int64_t b) { return a > 0 ? (a + b - 1) / b : 0; }
  void flat(int64_t &stride, int64_t n) {
    if (n <= 1) stride = 0;
    if (stride < 0) base += (n - 1) * stride, stride = -stride;
  }
};

// Whether two share a byte (interleaved ones do not).
inline bool overlap(const Lattice &a, const Lattice &b) {
  if (a.rows < 1 || a.heads < 1 || b.rows < 1 || b.heads < 1 || a.base >= b.end() || b.base >= a.end()) return false;
  // The distances from a piece of one to a piece of the other, of whole rows where the heads' strides differ.
  auto near = [](const Lattice &x, const Lattice &y) {
    const int64_t back = (x.rows - 1) * y.row + (x.heads - 1) * y.head;
    const Lattice between((const void *)(uintptr_t)(y.base - x.base - back), y.row, y.head, x.rows + y.rows - 1,
                          x.heads + y.heads - 1, 1);
    return between.meets(1 - y.width, x.width);
  };
  auto same = [](int64_t s, int64_t n, int64_t t, int64_t m) { return n == 1 || m == 1 || s == t; };
  auto with = [](Lattice x, const Lattice &y) {  // (a stride over one row says nothing)
    if (x.rows == 1) x.row = y.row;
    if (x.heads == 1) x.head = y.head;
    return x;
  };
  auto whole = [](Lattice x) {
    x.width += (x.heads - 1) * x.head;
    x.head = 0, x.heads = 1;
    return x;
  };
  if (same(a.row, a.rows, b.row, b.rows)) {
    if (same(a.head, a.heads, b.head, b.heads)) return near(with(a, b), with(b, a));
    const Lattice x = whole(a), y = whole(b);
    if (!near(with(x, y), with(y, x))) return false;
  }
  for (int64_t i = 0; i < a.rows; ++i)
    for (int64_t j = 0; j < a.heads; ++j) {
      const int64_t at = a.base + i * a.row + j * a.head;
      if (b.meets(at, at + a.width)) return true;
    }
  return false;
}

}  // namespace l20la

#endif  // L20_OVERLAP_H_
