// What the operators on device buffers share on the host: the refusal of a call, the device it runs on, the launch.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <new>
#include <stdexcept>
#include <string>

#include "../../include/c0ven_moe.h"

namespace c0ven {

std::string &open_error();  // moe_last_error(null)'s message, the calling thread's

struct OpError : std::runtime_error {
  moe_status st;
  OpError(moe_status s, const char *m) : std::runtime_error(m), st(s) {}
  OpError(moe_status s, const std::string &m) : std::runtime_error(m), st(s) {}
};

inline void op_require(bool ok, const char *why) {
  if (!ok) throw OpError(MOE_BAD_ARGUMENT, why);
}
inline void op_check(hipError_t e, const char *what) {
  if (e == hipSuccess) return;
  (void)hipGetLastError();  // (this call's error is not the next one's)
  throw OpError(MOE_ERROR, std::string(what) + ": " + hipGetErrorString(e));
}

// An operator's call: f checks and launches; what it throws becomes the status and the message.
template <typename F>
moe_status op_guarded(F f) {
  try {
    f();
    open_error().clear();
    return MOE_OK;
  } catch (const OpError &e) {
    open_error() = e.what();
    return e.st;
  } catch (const std::bad_alloc &) {
    return MOE_ERROR;
  } catch (const std::exception &e) {
    open_error() = e.what();
    return MOE_ERROR;
  }
}

// The host thread's device while an operator launches; the one before is set again after it.
class OnDevice {
 public:
  explicit OnDevice(int32_t device) {
    op_check(hipGetDevice(&before_), "hipGetDevice");
    if (before_ != device) {
      op_check(hipSetDevice(device), "hipSetDevice");
      other_ = true;
    }
  }
  ~OnDevice() {
    if (other_) (void)hipSetDevice(before_);
  }
  OnDevice(const OnDevice &) = delete;

 private:
  int before_ = 0;
  bool other_ = false;
};

// A launch that reports its own error and no earlier one's.
template <typename... P, typename... A>
void op_launch_lds(void (*kernel)(P...), uint64_t blocks, uint32_t threads, uint32_t lds, void *stream, A... args) {
  op_require(blocks <= 0xffffffffull / threads, "too many rows");  // (a launch has less than 2^32 threads)
  if (!blocks) return;
  static_assert(sizeof...(P) == sizeof...(A), "a kernel's arguments");
  [&](P... a) {
    void *list[] = {(void *)&a...};
    op_check(hipLaunchKernel((const void *)kernel, dim3((uint32_t)blocks), dim3(threads), list, lds, (hipStream_t)stream),
             "launch");
  }(args...);
}

template <typename... P, typename... A>
void op_launch(void (*kernel)(P...), uint64_t blocks, uint32_t threads, void *stream, A... args) {
  op_launch_lds(kernel, blocks, threads, 0, stream, args...);
}

inline bool op_float(uint32_t t) { return t == QT_F32 || t == QT_F16 || t == QT_BF16; }
inline uint32_t op_size(uint32_t t) { return t == QT_F32 ? 4 : 2; }
inline bool op_aligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// A dense buffer's rows: a pointer to whole elements (of no rows: null too) and a stride that holds a row.
inline void op_rows(const void *p, uint64_t stride, uint32_t rows, uint32_t cols, uint32_t type) {
  op_require(op_float(type), "the element type must be QT_F32, QT_F16 or QT_BF16");
  op_require(p || !rows, "null argument");
  op_require(op_aligned(p, op_size(type)), "a buffer must be aligned to its elements");
  op_require(stride >= cols && stride <= (1ull << 40), "a stride must hold a row");
}

}  // namespace c0ven
