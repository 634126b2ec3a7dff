// Memory of a call's arguments, compared on the host: outputs may not lie over inputs (other workgroups still read them) nor
// over each other.  Column slices of the same wider rows interleave in memory without sharing any of it, so base addresses
// and byte ranges alone do not tell.
#pragma once
#include "common.h"
#include <numeric>

namespace mmb {

struct Region {                                   // `rows` rows of `width` bytes, `ld` bytes apart; at == 0: no argument
  uintptr_t at;
  int64_t rows, width, ld;
};
inline Region row_region(const void* p, int64_t rows, int64_t width, int64_t ld, int es) { return {(uintptr_t)p, rows, width * es, ld * es}; }
inline Region flat_region(const void* p, int64_t bytes) { return {(uintptr_t)p, 1, bytes, bytes}; }

inline bool regions_meet(Region a, Region b) {
  if (!a.at || !b.at || a.width <= 0 || b.width <= 0) return false;
  auto end = [](const Region& r) { return (__int128)r.at + (__int128)(r.rows - 1) * r.ld + r.width; };
  if (end(a) <= (__int128)b.at || end(b) <= (__int128)a.at) return false;
  if (a.rows == 1 && b.rows == 1) return true;
  if (a.rows == 1) a.ld = b.ld;                   // (a single row's distance to the next means nothing)
  if (b.rows == 1) b.ld = a.ld;
  // columns modulo the common period: apart there, apart everywhere
  const int64_t period = std::gcd(a.ld, b.ld);
  const int64_t off = b.at >= a.at ? (int64_t)((b.at - a.at) % period) : (period - (int64_t)((a.at - b.at) % period)) % period;
  if (a.width <= off && off + b.width <= period) return false;
  if (a.rows > b.rows) std::swap(a, b);           // else row by row of the shorter one
  for (int64_t i = 0; i < a.rows; ++i) {
    const __int128 lo = (__int128)a.at + (__int128)i * a.ld, hi = lo + a.width;
    const __int128 past = lo - b.at - b.width;    // the first row of b that ends behind lo
    const __int128 j = past < 0 ? 0 : past / b.ld + 1;
    if (j < b.rows && (__int128)b.at + j * b.ld < hi) return true;
  }
  return false;
}

inline int check_apart(const char* who, const Region* outs, int no, const Region* ins, int ni) {
  for (int i = 0; i < no; ++i) {
    for (int j = 0; j < ni; ++j) MMB_REQUIRE(!regions_meet(outs[i], ins[j]), "%s: an output is the same memory as an input, or overlaps it", who);
    for (int j = 0; j < i; ++j) MMB_REQUIRE(!regions_meet(outs[i], outs[j]), "%s: two outputs are the same memory, or overlap", who);
  }
  return MMB_OK;
}

}  // namespace mmb
