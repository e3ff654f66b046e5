// What the files of the native host path share: views of tensors, error codes, scratch memory from torch's allocator.
#pragma once
#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/variable.h>

#include <limits>

#include "aotriton_amd/flash.h"

namespace fa_host {

using at::Tensor;

// ---- views ------------------------------------------------------------------------------------

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return FA_DTYPE_FLOAT32;
    case at::kHalf: return FA_DTYPE_FLOAT16;
    case at::kBFloat16: return FA_DTYPE_BFLOAT16;
    case at::kChar: return FA_DTYPE_INT8;
    case at::kShort: return FA_DTYPE_INT16;
    case at::kInt: return FA_DTYPE_INT32;
    case at::kLong: return FA_DTYPE_INT64;
    case at::kByte: return FA_DTYPE_UINT8;
    case at::kUInt16: return FA_DTYPE_UINT16;
    case at::kUInt32: return FA_DTYPE_UINT32;
    case at::kUInt64: return FA_DTYPE_UINT64;
    default: return FA_DTYPE_UNKNOWN;
  }
}

// View of a tensor of rank N (fa_tensor4, fa_tensor2 or fa_tensor1), null for an undefined one.
// False: not a view the operators take (rank, last stride, element type).
template <typename V, int N>
bool view_of(const Tensor& t, V* v) {
  *v = V{};
  if (!t.defined()) return true;
  if (t.dim() != N || t.stride(-1) != 1) return false;
  v->ptr = t.data_ptr();
  for (int i = 0; i < N; ++i) {
    v->sizes[i] = (uint64_t)t.size(i);
    v->strides[i] = (uint64_t)t.stride(i);
  }
  v->dtype = dtype_code(t.scalar_type());
  return v->dtype != FA_DTYPE_UNKNOWN;
}
inline bool view4(const Tensor& t, fa_tensor4* v) { return view_of<fa_tensor4, 4>(t, v); }
inline bool view2(const Tensor& t, fa_tensor2* v) { return view_of<fa_tensor2, 2>(t, v); }
// a rank-1 view has two elements or more: one element or none is a device scalar
inline bool view1(const Tensor& t, fa_tensor1* v) {
  return view_of<fa_tensor1, 1>(t, v) && (!t.defined() || t.numel() > 1);
}
inline bool view0(const Tensor& t, fa_tensor0* v) {
  *v = fa_tensor0{};
  if (!t.defined()) return true;
  if (t.dim() != 1 || t.numel() > 1) return false;
  v->ptr = t.data_ptr();
  v->dtype = dtype_code(t.scalar_type());
  return v->dtype != FA_DTYPE_UNKNOWN;
}

inline fa_tensor0 scalar_at(const Tensor& block, int i) {
  fa_tensor0 v{};
  v.ptr = static_cast<uint64_t*>(block.data_ptr()) + i;
  v.dtype = FA_DTYPE_UINT64;
  return v;
}

// The kernels move rows in aligned 16-byte pieces; a tensor whose rows are not made of them is copied.
inline Tensor pieces(const Tensor& t) {
  bool ok = t.stride(-1) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
  for (int64_t i = 0; ok && i + 1 < t.dim(); ++i) ok = t.size(i) <= 1 || t.stride(i) % 8 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

inline int32_t as_int32(int64_t x, const char* what) {
  TORCH_CHECK_VALUE(x >= 0 && x <= std::numeric_limits<int32_t>::max(), what, " must be a number of 31 bits, not ", x);
  return (int32_t)x;
}

inline void* current_stream() { return c10::hip::getCurrentHIPStream().stream(); }

inline const char* error_name(int rc) {
  switch (rc) {
    case 1: return "hipErrorInvalidValue";
    case 2: return "hipErrorOutOfMemory";
    case 13: return "hipErrorInvalidSymbol";
    case 209: return "hipErrorNoBinaryForGpu";
    case 217: return "hipErrorPeerAccessUnsupported";
    case 700: return "hipErrorIllegalAddress";
    case 801: return "hipErrorNotSupported";
    default: return "hipError";
  }
}

inline void check_rc(int rc, bool backend_is_not_implemented) {
  if (rc == FA_SUCCESS) return;
  TORCH_CHECK_NOT_IMPLEMENTED(!(backend_is_not_implemented && rc == FA_ERROR_PEER_ACCESS_UNSUPPORTED),
                              "backend cannot take this input");
  TORCH_CHECK(false, "flash operator failed: <hipError_t.", error_name(rc), ": ", rc, ">");
}

// Scratch memory of a forward, from torch's allocator: ordered with the stream, and a graph's own under capture.
// It is taken on the current device, whose current stream the call runs on: on another device (where the
// caller's tensors lie, say) the allocator could hand it on before the kernels are done with it.
struct Scratch {
  fa_allocator c{};
  Tensor held;
  Scratch() {
    c.cookie = this;
    c.alloc = &alloc;
  }
  static void* alloc(fa_allocator* self, uint64_t bytes) {
    auto* me = static_cast<Scratch*>(self->cookie);
    try {
      const at::Device device(at::kCUDA, c10::hip::current_device());
      me->held = at::empty({(int64_t)bytes}, at::TensorOptions(at::kByte).device(device));
      return me->held.data_ptr();
    } catch (...) {
      return nullptr;
    }
  }
};

// There is no forward-mode formula.  A call without a gradient goes past the Function, whose own error would
// come after the launch: without this check such a call would answer without the tangent.
inline void refuse_tangents(std::initializer_list<const Tensor*> inputs) {
  if (torch::autograd::ForwardADLevel::try_get_by_idx(0) == nullptr) return;      // (the tensors' own look takes locks)
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(),
                                "forward-mode AD of the attention operators (jvp) is not implemented");
}
}  // namespace fa_host
