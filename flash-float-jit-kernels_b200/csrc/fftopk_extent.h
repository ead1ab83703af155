// Where rows of strided arrays lie: host code without CUDA, which g++ compiles by itself.
#pragma once
#include <stdint.h>

namespace fftopk {

using Wide = __int128;  // (numbers of rows times strides, whatever a caller hands in)

// c * step for the whole numbers c in [lo, hi]
struct Steps {
  Wide step, lo, hi;
};

inline Wide floor_div(Wide a, Wide b) { return a / b - (a % b != 0 && (a < 0) != (b < 0)); }

// Is there a sum of x and one element of each of n Steps in [lo, hi]? Of the first one's elements those are tried that the others can bring into
// [lo, hi]: with the longest steps in front, hardly any where rows lie side by side.
inline bool reaches(const Steps* t, int n, Wide x, Wide lo, Wide hi) {
  if (n == 0) return lo <= x && x <= hi;
  Wide least = 0, most = 0, first_least = 0, first_most = 0;
  for (int i = n - 1; i >= 0; --i) {
    if (t[i].lo > t[i].hi) return false;
    least += first_least, most += first_most;
    const Wide a = t[i].step * t[i].lo, b = t[i].step * t[i].hi;
    first_least = a < b ? a : b, first_most = a < b ? b : a;
  }
  if (x + first_most + most < lo || x + first_least + least > hi) return false;
  if (t->step == 0) return reaches(t + 1, n - 1, x, lo, hi);
  // least element + most >= lo, and element + least <= hi
  const Wide from = lo - most - x, upto = hi - least - x, s = t->step;
  Wide a = s > 0 ? -floor_div(-from, s) : -floor_div(-upto, s), z = s > 0 ? floor_div(upto, s) : floor_div(from, s);
  if (a < t->lo) a = t->lo;
  if (z > t->hi) z = t->hi;
  if (n == 1) return a <= z;
  for (; a <= z; ++a)
    if (reaches(t + 1, n - 1, x + a * s, lo, hi)) return true;
  return false;
}

// No row of `width` elements - row (s, h) of `seqs` times `heads` begins at s * seq + h * head - lies on another one, as it would in a broadcast view,
// or where one stride is less than what the other one's rows take up. Rows in between others are fine.
inline bool rows_apart(int64_t seqs, int64_t seq, int64_t heads, int64_t head, int64_t width) {
  if (seqs <= 0 || heads <= 0 || width <= 0) return true;
  const Wide s = seq < 0 ? -(Wide)seq : (Wide)seq, h = head < 0 ? -(Wide)head : (Wide)head;
  if ((seqs > 1 && s < width) || (heads > 1 && h < width)) return false;
  if (seqs == 1 || heads == 1) return true;
  const bool seq_long = s >= h;
  if (seq_long ? (heads - 1) * h + width <= s : (seqs - 1) * s + width <= h) return true;
  // (the difference of two rows of different s and h; of equal ones it is a stride's multiple, see above)
  const Steps by_seq = {s, 1, (Wide)seqs - 1}, by_head = {-h, 1, (Wide)heads - 1};
  const Steps t[2] = {seq_long ? by_seq : by_head, seq_long ? by_head : by_seq};
  return !reaches(t, 2, 0, 1 - (Wide)width, (Wide)width - 1);
}

// Has a row of `a` an element in common with a row of `b`? Both are seqs times heads rows of `width` elements of `bytes` each, at strides of their own (in
// elements); rows in between the other one's are fine.
inline bool rows_meet(const void* a, int64_t a_seq, int64_t a_head, const void* b, int64_t b_seq, int64_t b_head, int64_t seqs, int64_t heads, int64_t width,
                      int bytes) {
  if (seqs <= 0 || heads <= 0 || width <= 0) return false;
  Steps t[4];
  int n = 0;
  auto add = [&](int64_t step, Wide lo, Wide hi) {  // (the longest in front)
    int i = n++;
    const Wide s = (Wide)step * bytes, abs = s < 0 ? -s : s;
    for (; i > 0 && (t[i - 1].step < 0 ? -t[i - 1].step : t[i - 1].step) < abs; --i) t[i] = t[i - 1];
    t[i] = {s, lo, hi};
  };
  auto both = [&](int64_t rows, int64_t of_a, int64_t of_b) {
    if (of_a == of_b) return add(of_a, 1 - (Wide)rows, (Wide)rows - 1);
    add(of_b, 0, (Wide)rows - 1);
    add(of_a, 1 - (Wide)rows, 0);
  };
  if (seqs > 1) both(seqs, a_seq, b_seq);  // (the stride of a lone one says nothing)
  if (heads > 1) both(heads, a_head, b_head);
  const Wide from = (Wide)reinterpret_cast<uintptr_t>(b) - (Wide)reinterpret_cast<uintptr_t>(a), row = (Wide)width * bytes;
  return reaches(t, n, from, 1 - row, row - 1);
}

}  // namespace fftopk
