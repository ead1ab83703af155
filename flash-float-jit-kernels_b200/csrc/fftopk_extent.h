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
  Wide least = 0, most = 0;
  for (int i = 1; i < n; ++i) {
    const Wide a = t[i].step * t[i].lo, b = t[i].step * t[i].hi;
    least += a < b ? a : b, most += a < b ? b : a;
  }
  if (t->lo > t->hi) return false;
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

}  // namespace fftopk
