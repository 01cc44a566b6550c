// Whether strided rows share memory (host code; the C entries and the torch module refuse outputs
// over what they are computed from).
#pragma once

#include <cstdint>

namespace qd {

// `n` rows of `bytes`, `stride` bytes apart.
struct Rows {
  const void* at;
  int64_t n, bytes, stride;
};

// Whether no byte is in both: their ranges lie apart, or rows of one stride lie beside each other.
inline bool apart(Rows a, Rows b) {
  if (a.n == 0 || b.n == 0 || a.bytes == 0 || b.bytes == 0) return true;
  const int64_t pa = (int64_t)reinterpret_cast<uintptr_t>(a.at), pb = (int64_t)reinterpret_cast<uintptr_t>(b.at);
  if (pa + (a.n - 1) * a.stride + a.bytes <= pb || pb + (b.n - 1) * b.stride + b.bytes <= pa) return true;
  if (a.n == 1) a.stride = b.stride;
  if (b.n == 1) b.stride = a.stride;
  if (a.stride != b.stride || a.n + b.n == 2) return false;
  const int64_t d = ((pb - pa) % a.stride + a.stride) % a.stride;  // from a row of a to the next of b
  return d >= a.bytes && d + b.bytes <= a.stride;
}

}  // namespace qd
