// What the operator registrations share: dtype enums, status and device checks, the stream, and the device error
// word of earlier kernels.
#pragma once
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <mutex>

#include "b200q.h"

namespace b200q_torch {

using at::Tensor;
using c10::optional;

inline int dtype_enum(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return B200Q_BF16;
    case at::kHalf: return B200Q_F16;
    case at::kFloat: return B200Q_F32;
    case at::kChar: return B200Q_I8;
    case at::kInt: return B200Q_I32;
    case at::kLong: return B200Q_I64;
    default: return 99;
  }
}

inline void check_status(int status, const char* op) {
  TORCH_CHECK(status == B200Q_OK, op, ": ", b200q_last_error(), " (", b200q_status_string(status), ")");
}

// A kernel that gives up a bounded wait returns early and leaves its output unfinished.  The library mirrors
// the device's error word into pinned host memory, so every operator call can look at it for free and raise
// (the error belongs to an earlier launch on this device; like the reference, which reports asynchronous
// launch failures at the next call, torch_npu/csrc/framework/OpParamMaker.cpp:258-264).  The mirror is set up
// on the first operator call on a device.
inline void surface_device_error(const char* op, const Tensor& t) {
  static std::once_flag once[64];
  const int dev = t.device().index();
  if (dev >= 0 && dev < 64) std::call_once(once[dev], [] { b200q_enable_host_error_word(); });
  const unsigned int code = b200q_peek_device_error();
  if (code != 0) {
    unsigned int seen = 0;
    b200q_device_error(&seen, 1);      // synchronises and clears, so that the next call can proceed
    TORCH_CHECK(code != 0x202, op, ": an earlier npu_moe_token_permute on ", t.device(),
                " met an expert index of 1024 or more (device error code 0x202); its output is incomplete");
    TORCH_CHECK(code != 0x203, op, ": an earlier gradient of npu_moe_token_unpermute on ", t.device(),
                " met a row that sorted_indices names twice (device error code 0x203); its output is wrong");
    TORCH_CHECK(false, op, ": an earlier kernel on ", t.device(), " gave up a bounded wait (device error code 0x", std::hex,
                code, "); its output is incomplete");
  }
}

// Same rule and message as the reference's generated wrapper (torchnpugen/custom_functions.py:137-208;
// expected text in test/custom_ops/test_npu_anti_quant.py:86-88).
inline void check_same_device(const char* op, const Tensor& first, std::initializer_list<const optional<Tensor>*> rest) {
  for (const optional<Tensor>* t : rest) {
    if (t->has_value() && (*t)->defined()) {
      TORCH_CHECK((*t)->device() == first.device(), op,
                  ": Expected all tensors to be on the same device, but found at least two devices, ",
                  first.device(), " and ", (*t)->device(), "!");
    }
  }
}

inline void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

}  // namespace b200q_torch
