// ilqr_overlap.h -- whether evenly spaced segments of memory meet (host code).
#ifndef ILQR_OVERLAP_H
#define ILQR_OVERLAP_H

#include <algorithm>
#include <cstdint>
#include <numeric>

namespace ilqr {

struct Every {
  int64_t count, stride;  // in bytes, not negative
};

// Runs of len bytes at base + sum of i_k stride_k, 0 <= i_k < count_k.
struct Strided {
  uintptr_t base;
  int64_t len;
  const Every* dims;
  int n;
  bool empty() const {
    for (int k = 0; k < n; ++k)
      if (dims[k].count < 1) return true;
    return len < 1;
  }
  uintptr_t hi() const {
    int64_t end = len;
    for (int k = 0; k < n; ++k) end += (dims[k].count - 1) * dims[k].stride;
    return base + (uintptr_t)end;
  }
};

// Two sets meet where the distance of a run of the one from a run of the other,
//   d = (b.base - a.base) + sum of x_k s_k,  lo_k <= x_k <= hi_k,
// lies strictly between -b.len and a.len; a stride that both have is one s_k
// (x counts the steps of b less those of a). The search goes through the strides
// from the largest down and takes of each only the x from which the smaller ones
// can still reach that interval: two or three where the stride steps over what
// they span, as in every array that is cut into columns, and the smallest stride
// is settled by a division.
class Meeting {
 public:
  // False only where no byte is in both.
  static bool of(const Strided& a, const Strided& b) {
    if (a.empty() || b.empty() || a.hi() <= b.base || b.hi() <= a.base) return false;
    Meeting m;
    m.above_ = -b.len;
    m.below_ = a.len;
    if (!m.add(a, -1) || !m.add(b, 1)) return true;
    while (m.merge_one()) {}
    std::sort(m.s_, m.s_ + m.n_, [](const Step& x, const Step& y) { return x.stride > y.stride; });
    m.min_[m.n_] = m.max_[m.n_] = m.measure_[m.n_] = 0;
    for (int k = m.n_ - 1; k >= 0; --k) {
      m.min_[k] = m.min_[k + 1] + m.s_[k].lo * m.s_[k].stride;
      m.max_[k] = m.max_[k + 1] + m.s_[k].hi * m.s_[k].stride;
      m.measure_[k] = std::gcd(m.measure_[k + 1], m.s_[k].stride);
    }
    return m.reach(0, (int64_t)(b.base - a.base));
  }

 private:
  struct Step {
    int64_t stride, lo, hi;
  };
  static constexpr int MAX_STEPS = 16;
  Step s_[MAX_STEPS];
  int64_t min_[MAX_STEPS + 1], max_[MAX_STEPS + 1], measure_[MAX_STEPS + 1];  // of the steps from k on
  int64_t above_ = 0, below_ = 0;
  int n_ = 0;
  int tries_ = 1 << 16;  // beyond them, and beyond MAX_STEPS, the answer is yes

  bool add(const Strided& r, int sign) {
    for (int k = 0; k < r.n; ++k) {
      const int64_t last = r.dims[k].count - 1, stride = r.dims[k].stride;
      if (last == 0 || stride == 0) continue;
      int at = 0;
      while (at < n_ && s_[at].stride != stride) ++at;
      if (at == n_) {
        if (n_ == MAX_STEPS) return false;
        s_[n_++] = Step{stride, 0, 0};
      }
      if (sign > 0) s_[at].hi += last;
      else s_[at].lo -= last;
    }
    return true;
  }

  // A stride of r smaller ones, whose own x fill the steps between its: together
  // they take every multiple of the smaller stride in their range.
  bool merge_one() {
    for (int i = 0; i < n_; ++i)
      for (int j = 0; j < n_; ++j) {
        const int64_t r = s_[i].stride / s_[j].stride;
        if (i == j || r * s_[j].stride != s_[i].stride || s_[j].hi - s_[j].lo < r - 1) continue;
        s_[j].lo += r * s_[i].lo;
        s_[j].hi += r * s_[i].hi;
        s_[i] = s_[--n_];
        return true;
      }
    return false;
  }

  static int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0 ? 1 : 0); }  // b > 0

  bool reach(int k, int64_t d) {
    if (k == n_) return d > above_ && d < below_;
    // the first distance above the lower end that differs from d by whole measures
    const int64_t off = (d - above_ - 1) % measure_[k];
    if (above_ + 1 + off + (off < 0 ? measure_[k] : 0) >= below_) return false;
    const Step& s = s_[k];
    const int64_t first = std::max(s.lo, floor_div(above_ - d - max_[k + 1], s.stride) + 1);
    const int64_t last = std::min(s.hi, -floor_div(-(below_ - d - min_[k + 1]), s.stride) - 1);
    if (k + 1 == n_) return first <= last;
    for (int64_t x = first; x <= last; ++x)
      if (--tries_ < 0 || reach(k + 1, d + x * s.stride)) return true;
    return false;
  }
};

}  // namespace ilqr

#endif
