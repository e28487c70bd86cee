// What the C entries of the operators check of their arguments, on the host, before anything is launched.
#pragma once
#include <hip/hip_runtime.h>

#include <stdexcept>
#include <string>

#include "../../include/tts_hip.h"

namespace tts {

tts_status report(tts_status st, const std::string &msg);  // runtime.hip: sets tts_last_error

struct Refused : std::runtime_error {
  tts_status status;
  Refused(tts_status st, const std::string &msg) : std::runtime_error(msg), status(st) {}
};

[[noreturn]] inline void invalid(const std::string &msg) { throw Refused(TTS_INVALID, msg); }
[[noreturn]] inline void unsupported(const std::string &msg) { throw Refused(TTS_UNSUPPORTED, msg); }

inline int64_t item_size(int dtype) { return dtype == TTS_I8 ? 1 : dtype == TTS_F16 || dtype == TTS_BF16 ? 2 : 4; }
inline const char *type_name(int dtype) {
  static const char *names[] = {"f32", "f16", "bf16", "i8", "i32"};
  return dtype >= 0 && dtype < 5 ? names[dtype] : "an unknown type";
}

constexpr int64_t MOST_SIZE = (int64_t)1 << 30;  // of a dimension: sums of two fit 32 bits

// one argument of a call, by its name
struct Arg {
  const tts_tensor *t;
  std::string name;
  Arg(const tts_tensor *tensor, const char *n) : t(tensor), name(n) {
    if (!t) invalid(name + " is missing");
    if (t->dtype < TTS_F32 || t->dtype > TTS_I32) invalid(name + " has an unknown type");
    if (t->rank < 1 || t->rank > 3) invalid(name + " has " + std::to_string(t->rank) + " dimensions");
    for (int d = 0; d < t->rank; d++) {
      if (t->shape[d] < 0 || t->shape[d] > MOST_SIZE) invalid(name + ": dimension " + std::to_string(d) + " is " + std::to_string(t->shape[d]));
      if (t->stride[d] < 0 || t->stride[d] > ((int64_t)1 << 48)) invalid(name + ": stride " + std::to_string(d) + " is " + std::to_string(t->stride[d]));
    }
    if ((uintptr_t)t->ptr % item_size(t->dtype)) invalid(name + " is not aligned to its elements");
  }
  int64_t size(int d) const { return t->shape[d]; }
  int64_t stride(int d) const { return t->stride[d]; }
  Arg &rank(int n) {
    if (t->rank != n) invalid(name + " has " + std::to_string(t->rank) + " dimensions, not " + std::to_string(n));
    return *this;
  }
  Arg &type(int want) {
    if (t->dtype != want) invalid(name + " is " + type_name(t->dtype) + ", not " + type_name(want));
    return *this;
  }
  Arg &shape(int d, int64_t want, const char *like) {
    if (size(d) != want) invalid(name + ": dimension " + std::to_string(d) + " is " + std::to_string(size(d)) + ", but " + like + " says " + std::to_string(want));
    return *this;
  }
  Arg &neighbours() {  // the elements of a row
    const int d = t->rank - 1;
    if (stride(d) != 1 && size(d) > 1) invalid(name + ": its last dimension has stride " + std::to_string(stride(d)) + ", not 1");
    return *this;
  }
  Arg &some(int d) {
    if (size(d) < 1) invalid(name + ": dimension " + std::to_string(d) + " is empty");
    return *this;
  }
  // nothing in it is there twice (for what is written; its last dimension has stride 1)
  Arg &distinct() {
    if (t->rank == 2 && size(0) > 1 && stride(0) < size(1)) invalid(name + ": its rows overlap");
    if (t->rank == 3) {
      auto nested = [&](int outer, int inner) {
        const int64_t row = size(2), rows = size(inner) > 1 ? (size(inner) - 1) * stride(inner) + row : row;
        return (size(inner) <= 1 || stride(inner) >= row) && (size(outer) <= 1 || stride(outer) >= rows);
      };
      if (!empty() && !nested(0, 1) && !nested(1, 0)) invalid(name + ": its rows overlap");
    }
    return *this;
  }
  bool empty() const {
    for (int d = 0; d < t->rank; d++)
      if (size(d) == 0) return true;
    return false;
  }
  void present() const {
    if (!t->ptr && !empty()) invalid(name + " is a null pointer");
  }
  uintptr_t first() const { return (uintptr_t)t->ptr; }
  uintptr_t end() const {  // the byte behind its last element
    int64_t last = 0;
    for (int d = 0; d < t->rank; d++) last += (size(d) - 1) * stride(d);
    return first() + (uintptr_t)(last + 1) * item_size(t->dtype);
  }
};

// whether they share memory: by their extents, except that columns of one buffer with rows of the same distance are told apart
inline bool overlap(const Arg &a, const Arg &b) {
  if (a.empty() || b.empty() || a.end() <= b.first() || b.end() <= a.first()) return false;
  if (a.t->rank >= 2 && b.t->rank >= 2 && item_size(a.t->dtype) == item_size(b.t->dtype) && a.stride(0) == b.stride(0) && a.stride(0) > 0) {
    auto width = [](const Arg &x) {  // of the columns that a row takes
      int64_t last = 0;
      for (int d = 1; d < x.t->rank; d++) last += (x.size(d) - 1) * x.stride(d);
      return last + 1;
    };
    const int64_t item = item_size(a.t->dtype), pitch = a.stride(0) * item;
    const int64_t apart = ((int64_t)(b.first() - a.first()) % pitch + pitch) % pitch;
    if (apart >= width(a) * item && apart + width(b) * item <= pitch) return false;
  }
  return true;
}
inline void apart(const Arg &out, const Arg &in) {
  if (overlap(out, in)) invalid(out.name + " shares memory with " + in.name);
}

inline void half_type(const Arg &a) {
  if (a.t->dtype == TTS_F32) unsupported(a.name + " is f32: the operator takes f16 and bf16");
  if (a.t->dtype != TTS_F16 && a.t->dtype != TTS_BF16) invalid(a.name + " is " + std::string(type_name(a.t->dtype)) + ", not f16 or bf16");
}

inline void check_workspace(void *workspace, size_t bytes, size_t need) {
  if (bytes < need) invalid("the workspace has " + std::to_string(bytes) + " bytes, and " + std::to_string(need) + " are needed");
  if (need && !workspace) invalid("the workspace is a null pointer");
  if ((uintptr_t)workspace % 256) invalid("the workspace is not aligned to 256 bytes");
}

template <class F>
tts_status guarded(const char *who, F &&f) {
  try {
    const hipError_t e = f();
    return e == hipSuccess ? TTS_OK : report(TTS_HIP_ERROR, std::string(who) + ": " + hipGetErrorString(e));
  } catch (const Refused &e) {
    return report(e.status, std::string(who) + ": " + e.what());
  } catch (const std::exception &e) {
    return report(TTS_INVALID, std::string(who) + ": " + e.what());
  }
}

}  // namespace tts
