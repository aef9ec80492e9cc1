// Whether two operands of a call share a byte: rows of `row` bytes at `at` + i0 step[0] + i1 step[1] + i2
// step[2].  Views of one projection interleave without sharing any, so comparing their first and last
// bytes is not enough.
#pragma once

#include <stdint.h>

#include "asc_hip.h"

namespace asc {

struct Region {
  const char* name;
  uintptr_t at;
  int64_t size[3];
  int64_t step[3];
  int64_t row;  // 0: nothing
  __int128 first, end;  // of all bytes
};

inline Region spanned(Region r) {
  r.first = r.at;
  r.end = r.first + r.row;
  for (int i = 0; i < 3; ++i) {
    (r.step[i] < 0 ? r.first : r.end) += static_cast<__int128>(r.step[i]) * (r.size[i] - 1);
  }
  return r;
}

inline Region region_of(const char* name, const asc_rows_t& r, int64_t batch, int64_t heads, int64_t seq, int64_t row,
                        int64_t element) {
  const auto bytes = [&](int64_t stride, int64_t n) {  // a dimension of one element is not stepped over
    int64_t b = 0;
    return n > 1 && !__builtin_mul_overflow(stride, element, &b) ? b : (n > 1 ? INT64_MAX : 0);
  };
  const bool any = r.data != nullptr && batch > 0 && heads > 0 && seq > 0;
  return spanned({name,
                  reinterpret_cast<uintptr_t>(r.data),
                  {batch, heads, seq},
                  {bytes(r.batch_stride, batch), bytes(r.head_stride, heads), bytes(r.seq_stride, seq)},
                  any ? row * element : 0,
                  0,
                  0});
}
inline Region region_of(const char* name, const void* data, int64_t bytes) {
  return spanned({name, reinterpret_cast<uintptr_t>(data), {1, 1, 1}, {0, 0, 0}, data ? bytes : 0, 0, 0});
}

inline bool same_place(const Region& a, const Region& b) {
  for (int i = 0; i < 3; ++i) {
    if (a.size[i] != b.size[i] || a.step[i] != b.step[i]) return false;
  }
  return a.at == b.at && a.row == b.row;
}

// The distance from a row of `a` to a row of `b` is first + sum x_k step_k with each x_k in a range of its
// own (equal steps of both joined); they share bytes where it lies between -b.row and a.row.  The steps are
// tried from the largest down, each only as far as the rest can make up: one to three values each
// where the steps are those of one buffer.  Operands laid out so differently that this takes long are taken
// to overlap.
class OverlapSearch {
 public:
  OverlapSearch(const Region& a, const Region& b) : low_(-b.row), high_(a.row) {
    for (int i = 0; i < 3; ++i) {
      add(a.step[i], -(a.size[i] - 1), 0);
      add(b.step[i], 0, b.size[i] - 1);
    }
    for (int i = 1; i < n_; ++i) {
      for (int j = i; j > 0 && terms_[j].step > terms_[j - 1].step; --j) {
        const Term t = terms_[j];
        terms_[j] = terms_[j - 1];
        terms_[j - 1] = t;
      }
    }
    for (int i = n_ - 1; i >= 0; --i) {
      least_[i] = least_[i + 1] + terms_[i].first * terms_[i].step;
      most_[i] = most_[i + 1] + terms_[i].last * terms_[i].step;
    }
    found_ = search(0, static_cast<wide>(b.at) - static_cast<wide>(a.at));
  }
  bool found() const { return found_; }

 private:
  typedef __int128 wide;
  struct Term {
    wide step, first, last;
  };
  void add(int64_t step, int64_t first, int64_t last) {
    if (step == 0 || first == last) return;
    Term t{step, first, last};
    if (step < 0) t = {-static_cast<wide>(step), -static_cast<wide>(last), -static_cast<wide>(first)};
    for (int i = 0; i < n_; ++i) {
      if (terms_[i].step == t.step) {
        terms_[i].first += t.first;
        terms_[i].last += t.last;
        return;
      }
    }
    terms_[n_++] = t;
  }
  static wide floor_div(wide a, wide b) { return a / b - (a % b != 0 && a < 0 ? 1 : 0); }
  bool search(int k, wide at) {
    if (at + most_[k] <= low_ || at + least_[k] >= high_) return false;
    if (k == n_) return true;
    if (--left_ < 0) return true;
    const Term& t = terms_[k];
    wide x = floor_div(low_ - at - most_[k + 1], t.step) + 1, end = floor_div(high_ - 1 - at - least_[k + 1], t.step);
    if (x < t.first) x = t.first;
    if (end > t.last) end = t.last;
    for (; x <= end; ++x) {
      if (search(k + 1, at + x * t.step)) return true;
    }
    return false;
  }

  wide low_, high_;
  Term terms_[6];
  wide least_[7] = {}, most_[7] = {};
  int n_ = 0, left_ = 4096;
  bool found_ = false;
};

inline bool overlap(const Region& a, const Region& b) {
  return a.row != 0 && b.row != 0 && a.first < b.end && b.first < a.end && OverlapSearch(a, b).found();
}

}  // namespace asc
