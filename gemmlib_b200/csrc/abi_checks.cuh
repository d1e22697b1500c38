// What the extern "C" entry points of the 8-bit paths share: the checks of their arguments, and the way their errors go.
#pragma once

#include <cstddef>
#include <cstdint>
#include <exception>
#include <initializer_list>
#include <string>

#include "ms_blkq4gemm.h"

namespace blkq4 {
namespace abi {

inline int fail(void* err, const std::string& msg) {
  if (err) *reinterpret_cast<std::string*>(err) = msg;
  return -1;
}

// A matrix argument of `rows` rows of `cols` elements: empty if it is all there, else what is wrong with it.
inline std::string check_matrix(const char* name, const void* ptr, size_t size, int64_t ld, int rows, int cols, int elt) {
  if (!ptr) return std::string("Null tensor pointer: ") + name;
  if (reinterpret_cast<uintptr_t>(ptr) % elt != 0) return std::string("Misaligned tensor: ") + name;
  if (ld < cols && rows > 1)
    return std::string("Leading dimension of ") + name + " is smaller than its rows: " + std::to_string(ld);
  if (rows > 1 && ld > (INT64_MAX / 2 / elt - cols) / (rows - 1)) return std::string("Leading dimension of ") + name + " is out of range";
  const uint64_t need = ((uint64_t)(rows - 1) * (uint64_t)(rows > 1 ? ld : 0) + (uint64_t)cols) * (uint64_t)elt;
  if (size < need)
    return std::string("Unexpected size of ") + name + ": " + std::to_string(size) + " expected: " + std::to_string(need);
  return std::string();
}

inline std::string check_shape(int dtype, int rows, int cols) {
  if (dtype != INT8_FP16 && dtype != INT8_BF16) return "Unsupported type: " + std::to_string(dtype);
  if (rows <= 0 || cols <= 0) return "Empty problem size: " + std::to_string(rows) + "x" + std::to_string(cols);
  if (cols > (1 << 28)) return "Too many columns: " + std::to_string(cols);
  return std::string();
}

struct Matrix {
  const char* name;
  const void* ptr;
  size_t size;
  int64_t ld;
  int rows, cols, elt;
};

inline std::string check_all(std::initializer_list<Matrix> all) {
  for (const Matrix& m : all) {
    std::string e = check_matrix(m.name, m.ptr, m.size, m.ld, m.rows, m.cols, m.elt);
    if (!e.empty()) return e;
  }
  return std::string();
}

// One call: `check` and `launch` return an error text or nothing.  No exception leaves a C entry point.
template <class Check, class Launch>
int guarded(void* err, Check&& check, Launch&& launch) noexcept {
  try {
    std::string e = check();
    if (!e.empty()) return fail(err, e);
    e = launch();
    if (!e.empty()) return fail(err, "Kernel execution failed: " + e);
    return 0;
  } catch (const std::exception& x) {
    try {
      return fail(err, x.what());
    } catch (...) {
    }
  } catch (...) {
  }
  return -1;
}

// Rows of a matrix of one row follow one another at no distance: any ld will do.
inline int64_t row_pitch(int64_t ld, int rows, int cols) { return rows > 1 ? ld : (int64_t)((cols + 15) / 16) * 16; }

}  // namespace abi
}  // namespace blkq4
