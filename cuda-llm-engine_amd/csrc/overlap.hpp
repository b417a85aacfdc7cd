// Whether arrays of a call share memory: host arithmetic only (not exported).
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace llmk {

// n rows, ld elements of 2 bytes apart, of `pieces` pieces each, `apart` elements apart, of which a call takes the first
// `width`. A contiguous array is one row of one piece.
struct Rows {
  uintptr_t at;
  long long n, ld, pieces, apart, width;
  long long row() const { return (pieces - 1) * apart + width; }  // from a row's first element to its last
};
inline Rows rows_of(const void* p, long long n, long long ld, long long width) {
  return {reinterpret_cast<uintptr_t>(p), n, ld, 1, width, width};
}
inline Rows bytes_of(const void* p, size_t bytes) { return rows_of(p, 1, 0, (long long)((bytes + 1) / 2)); }

// Whether a row of a shares elements with one of b that begins `d` behind it. Their pieces are walked side by side.
inline bool pieces_overlap(const Rows& a, const Rows& b, long long d) {
  if (d >= a.row() || -d >= b.row()) return false;
  for (long long i = 0, j = 0; i < a.pieces && j < b.pieces;) {
    const long long x = i * a.apart, y = d + j * b.apart;
    if (x + a.width <= y) ++i;
    else if (y + b.width <= x) ++j;
    else return true;
  }
  return false;
}

// Whether a and b share elements. Nothing does with an array that is not there or of no elements. Rows are as long as ld
// at most, where there are two or more. Addresses are at least as aligned as elements.
inline bool overlap(const Rows& a, const Rows& b) {
  if (!a.at || !b.at || a.n <= 0 || b.n <= 0 || a.row() <= 0 || b.row() <= 0) return false;
  const long long d = ((long long)b.at - (long long)a.at) / 2;  // from a's first element to b's
  if (d >= (a.n - 1) * a.ld + a.row() || -d >= (b.n - 1) * b.ld + b.row()) return false;
  if (a.ld == b.ld && a.ld > 0) {  // columns of one matrix: b's row s lies over a's row s + k and may reach into the next
    const long long at = (d % a.ld + a.ld) % a.ld, k = (d - at) / a.ld;
    const auto there = [&](long long behind) { return behind > -b.n && behind < a.n; };
    return (there(k) && pieces_overlap(a, b, at)) || (there(k + 1) && pieces_overlap(a, b, at - a.ld));
  }
  for (long long i = 0, j = 0; i < a.n && j < b.n;) {  // both walked in order of their addresses
    const long long x = i * a.ld, y = d + j * b.ld;
    if (pieces_overlap(a, b, y - x)) return true;
    if (x + a.row() <= y + b.row()) ++i; else ++j;
  }
  return false;
}

}  // namespace llmk
