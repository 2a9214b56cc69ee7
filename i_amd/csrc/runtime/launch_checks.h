// What the launchers of the kernels beside the language's own path share: checks of arguments, launches, workspaces, errors.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <string>

#include "../../../include/i_attend.h"
#include "../core/error.h"
#include "hip_rt.h"

namespace ihip::host {

using ihip::Err;

constexpr int64_t kMaxGrid = 0x7fffffff;
constexpr int64_t kMaxThreads = 0xffffffff;  // of a launch along x
constexpr int64_t kMaxExtent = int64_t(1) << 30;

inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t element_bytes(int64_t dtype) { return dtype == I_DTYPE_BF16 ? 2 : 4; }
inline const char* type_name(int64_t dtype) { return dtype == I_DTYPE_BF16 ? "bf16" : "f32"; }

inline Err check_extent(const char* name, int64_t n) {
  if (n < 0 || n > kMaxExtent) return std::string(name) + " must be 0 .. 2^30, not " + std::to_string(n);
  return {};
}
inline Err check_common(int64_t dtype, int64_t b, int64_t hq, int64_t hkv, int64_t d, double scale, double cap) {
  if (dtype != I_DTYPE_F32 && dtype != I_DTYPE_BF16) return "unknown dtype";
  if (Err e = check_extent("b", b); !e.empty()) return e;
  if (hq < 1 || hkv < 1 || hq > 65535 || hq % hkv != 0) return "query heads must be a multiple of key heads (1 .. 65535), not " + std::to_string(hq) + " over " + std::to_string(hkv);
  if (b * hq > kMaxExtent) return "too many heads";
  if (d < 8 || d > 256 || d % 8 != 0) return "head size must be a multiple of 8 up to 256, not " + std::to_string(d);
  if (!std::isfinite(scale) || !std::isfinite((float)scale)) return "scale must be finite";
  if (!std::isfinite(cap) || !std::isfinite((float)cap) || cap < 0.0) return "cap must be finite and not negative (0: no cap)";
  if (cap > 0.0 && !std::isfinite((float)scale / (float)cap * 4.0f)) return "scale / cap is out of range";
  return {};
}

// A [b, h, n, d] operand whose rows are read and written in pieces of 16 bytes.
inline Err check_tensor(const char* name, const i_attend_tensor* t, int64_t dtype) {
  if (!t) return std::string(name) + " is missing";
  const int64_t e = (int64_t)element_bytes(dtype);
  if (!t->data) return std::string(name) + ": null device pointer";
  if ((uintptr_t)t->data % 16 != 0) return std::string(name) + " must start on a 16-byte boundary";
  for (int64_t s : {t->stride_b, t->stride_h, t->stride_n}) {
    if (s < 0) return std::string(name) + ": negative strides are not supported";
    if (s * e % 16 != 0) return std::string(name) + ": strides must be multiples of 16 bytes";
  }
  // (a tile of 64 rows is addressed from its first row in 32 bits)
  if (t->stride_n * e >= (int64_t(1) << 25)) return std::string(name) + ": rows more than 32 MiB apart are not supported";
  return {};
}

template <typename Params>
Err run(const std::string& name, ihip::CodeObject object, int64_t grid, unsigned threads, const Params& p, hipStream_t stream, unsigned across = 1) {
  if (grid > kMaxGrid) return name + ": grid too large";
  hipFunction_t fn;
  if (Err e = ihip::builtin_function(name.c_str(), &fn, object); !e.empty()) return e;
  return ihip::launch(fn, (unsigned)grid, across, 1, threads, &p, sizeof(p), stream);
}

// Carves temporaries out of the caller's workspace, or adds up what they take.
struct Carver {
  char* base;
  size_t at = 0;
  template <typename T>
  T* take(int64_t count) {
    T* here = base ? reinterpret_cast<T*>(base + at) : nullptr;
    at += (size_t)up(count * (int64_t)sizeof(T), 256);
    return here;
  }
};

inline Err check_workspace(void* workspace, size_t given, size_t needed) {
  if (needed == 0) return {};
  if (!workspace || given < needed) return "workspace of " + std::to_string(needed) + " bytes needed, " + std::to_string(workspace ? given : 0) + " given";
  if ((uintptr_t)workspace % 256 != 0) return "workspace must start on a 256-byte boundary";
  return {};
}

// Nothing is thrown across the C boundary.
template <typename F>
int guarded(const char* what, F&& call) {
  Err e;
  try {
    e = call();
  } catch (const std::exception& x) {
    e = x.what();
  } catch (...) {
    e = "unexpected failure";
  }
  if (e.empty()) return 0;
  icore::set_error(std::string(what) + ": " + e);
  return -1;
}

}  // namespace ihip::host
