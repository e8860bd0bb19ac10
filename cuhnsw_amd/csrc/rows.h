// Operators on tables of vectors that are in device memory: what the three files of kernels (rows_lookup.hip,
// rows_scores.hip, rows_select.hip) share, and the calls that the engine makes of them.
//
// Unlike the engine's calls these take device pointers and a stream, allocate nothing, wait for nothing and may be
// recorded into a graph: scratch memory is the caller's (each operator says how much it wants).
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>

#include "host_staging.h"  // HIP_CHECK

namespace cuhnsw_amd {

enum ElementType { TYPE_F32 = 0, TYPE_F16 = 1, TYPE_BF16 = 2 };
inline size_t element_size(int type) { return type == TYPE_F32 ? 4 : 2; }

struct bf16 {
  uint16_t bits;
};

__device__ inline float widen(float x) { return x; }
__device__ inline float widen(_Float16 x) { return (float)x; }
__device__ inline float widen(bf16 x) { return __uint_as_float((uint32_t)x.bits << 16); }
// to nearest, ties to even; NaN stays NaN
template <typename T>
__device__ inline T narrow(float x);
template <>
__device__ inline float narrow<float>(float x) { return x; }
template <>
__device__ inline _Float16 narrow<_Float16>(float x) { return (_Float16)x; }
template <>
__device__ inline bf16 narrow<bf16>(float x) {
  return bf16{__builtin_bit_cast(uint16_t, (__bf16)x)};  // (one instruction of the machine)
}

// n elements that move together (the widest such access that rows, strides and addresses allow is chosen per call)
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T at[N];
};

// the same at any address that fits the elements
template <typename T, int N>
struct LoosePack {
  T at[N];
};

// the message of the last call without an engine that failed in this thread (engine.hip)
void set_call_error(const char* message) noexcept;

// Body of a C entry point: no exception leaves it.
template <typename F>
int call_guarded(F&& f) noexcept {
  try {
    static const bool any_device = [] {
      int devices = 0;
      const bool there = hipGetDeviceCount(&devices) == hipSuccess && devices > 0;
      (void)hipGetLastError();
      return there;
    }();
    if (!any_device) {
      set_call_error("no HIP device available: this call needs a GPU");
      return -1;
    }
    f();
    set_call_error("");
    return 0;
  } catch (const std::exception& ex) {
    set_call_error(ex.what());
  } catch (...) {
    set_call_error("unknown error");
  }
  return -1;
}

inline void want(bool ok, const char* message) {
  if (!ok) throw std::runtime_error(message);
}
inline bool known_type(int type) { return type == TYPE_F32 || type == TYPE_F16 || type == TYPE_BF16; }

// Runs f with a null pointer of the element type: f((float*)nullptr) and so on.
template <typename F>
void with_type(int type, F&& f) {
  if (type == TYPE_F32) f((float*)nullptr);
  else if (type == TYPE_F16) f((_Float16*)nullptr);
  else f((bf16*)nullptr);
}

// Parts of a caller's workspace, one after the other; measures where there is no memory yet.
class WorkspaceParts {
 public:
  explicit WorkspaceParts(void* memory) : memory_(static_cast<unsigned char*>(memory)) {}
  template <typename T>
  T* part(size_t n) {
    T* p = memory_ ? reinterpret_cast<T*>(memory_ + used_) : nullptr;
    used_ += (n * sizeof(T) + 255) & ~(size_t)255;
    return p;
  }
  size_t used() const { return used_; }

 private:
  unsigned char* memory_;
  size_t used_ = 0;
};

struct LookupArgs {
  const void* table;
  int table_type;
  long long num_rows, row_stride;  // stride in elements
  int num_dims;
  const void* ids;
  int ids_64;
  long long num_ids;
  float scale;
  void* out;  // [num_ids, num_dims]
  int out_type;
};
void launch_lookup(const LookupArgs& a, hipStream_t stream);

struct PackArgs {
  const void* rows;
  int type;
  long long row_stride, num_rows;
  int num_dims, group;
  unsigned char* codes;  // [num_rows, 16 * ceil(num_dims / 32)]
  void *scales, *offsets;  // [num_rows, ceil(num_dims / group)]; offsets may be null
  int scale_type;
};
void launch_pack(const PackArgs& a, hipStream_t stream);

}  // namespace cuhnsw_amd
