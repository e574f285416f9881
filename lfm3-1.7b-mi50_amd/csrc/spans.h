// What the C entry points check their arguments with: memory that a call reads or writes, and whether pieces of it meet.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

namespace dspark {

// Compute units of the current device (queried once per device).
inline int device_cus() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (!n) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

inline bool on(const void* p, uintptr_t bytes) { return p && (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Memory that a call reads or writes: `rows` pieces of n bytes, `stride` apart (stride >= n); p NULL or n 0: none.
struct Span {
  const void* p;
  size_t n;
  size_t rows = 1, stride = 0;
};
// A piece of n bytes at `at` and some row of y share a byte: of y's rows the first that ends behind `at` begins before the piece ends.
inline bool meets(uintptr_t at, size_t n, const Span& y) {
  const uintptr_t b = reinterpret_cast<uintptr_t>(y.p);
  const size_t i = at < b + y.n ? 0 : y.rows > 1 ? (at - b - y.n) / y.stride + 1 : 1;
  return i < y.rows && b + i * y.stride < at + n;
}
inline bool overlap(const Span& x, const Span& y) {
  if (!x.p || !y.p || !x.n || !y.n) return false;
  const uintptr_t a = reinterpret_cast<uintptr_t>(x.p), b = reinterpret_cast<uintptr_t>(y.p);
  if (a >= b + (y.rows - 1) * y.stride + y.n || b >= a + (x.rows - 1) * x.stride + x.n) return false;
  if (x.rows > 1 && y.rows > 1 && x.stride == y.stride) {
    // row j = i + k of y meets row i of x where k stride is in (a - b - y.n, a - b + x.n): the least such k decides
    const int64_t s = (int64_t)x.stride, lo = (int64_t)a - (int64_t)b - (int64_t)y.n;
    const int64_t k = std::max((lo >= 0 ? lo / s : -((s - 1 - lo) / s)) + 1, -((int64_t)x.rows - 1));
    return k < (int64_t)y.rows && k * s < (int64_t)a - (int64_t)b + (int64_t)x.n;
  }
  if (x.rows > y.rows) return overlap(y, x);  // (few rows of one with many of the other: heads, tokens of a block)
  for (size_t i = 0; i < x.rows; ++i)
    if (meets(a + i * x.stride, x.n, y)) return true;
  return false;
}
// Nothing that is written shares a byte with what is read, nor with anything else that is written: workgroups read and store in
// no order among each other.
template <size_t NR, size_t NW>
inline bool apart(const Span (&reads)[NR], const Span (&writes)[NW]) {
  for (size_t i = 0; i < NW; ++i) {
    for (const Span& r : reads)
      if (overlap(r, writes[i])) return false;
    for (size_t j = 0; j < i; ++j)
      if (overlap(writes[j], writes[i])) return false;
  }
  return true;
}

}  // namespace dspark
