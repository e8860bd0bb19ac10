// Rows held in 4 bits with a scale for every group of elements, and products of queries with all of them.
//
//   w[n][k] = scale[n][k / group] * (code[n][k] - 8)                         without offsets
//   w[n][k] = scale[n][k / group] * code[n][k] + offset[n][k / group]        with offsets
//   out[m][n] = alpha * sum over k of w[n][k] * query[m][k]  (+ bias[n])
//
// A row's codes are 16 bytes for every 32 elements, element 2 i in the low half of byte i; what is behind the last element
// is not looked at.  Scales and offsets are float16 or bfloat16.
#include <algorithm>

#include "../../include/cuhnsw_amd.h"
#include "rows.h"

namespace cuhnsw_amd {

__device__ inline float half_bits(uint16_t bits, bool is_bf16) {
  return is_bf16 ? __uint_as_float((uint32_t)bits << 16) : (float)__builtin_bit_cast(_Float16, bits);
}

// ------------------------------------------------------------------------------------------------ packing
// Eight consecutive elements per lane, so a group is 4, 8 or 16 neighbouring lanes, whose extremes meet by shuffles.  The
// scale is rounded first and the codes are taken with the rounded one: what is stored is what is multiplied with.
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const T* rows, long long row_stride, long long num_rows, int num_dims, int group,
                                                   int lanes_per_row, unsigned char* codes, uint16_t* scales, uint16_t* offsets, int scale_bf16) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long n = i / lanes_per_row;
  const int l = (int)(i - n * lanes_per_row), first = 8 * l;
  const bool row_there = n < num_rows;
  float x[8], low = INFINITY, high = -INFINITY;
  for (int j = 0; j < 8; ++j) {
    const bool there = row_there && first + j < num_dims;
    x[j] = there ? widen(rows[n * row_stride + first + j]) : 0.f;
    if (there) {
      low = fminf(low, x[j]);
      high = fmaxf(high, x[j]);
    }
  }
  for (int step = 1; step < group / 8; step <<= 1) {
    low = fminf(low, __shfl_xor(low, step));
    high = fmaxf(high, __shfl_xor(high, step));
  }
  if (!row_there || first / group * group >= num_dims) return;
  const float most = scale_bf16 ? 3.3895314e38f : 65504.f;
  auto store = [&](float v) -> uint16_t {
    return scale_bf16 ? narrow<bf16>(v).bits : __builtin_bit_cast(uint16_t, (_Float16)v);
  };
  const uint16_t scale_bits = store(fminf(offsets ? high / 15.f - low / 15.f : fmaxf(high, -low) / 7.f, most));
  const uint16_t offset_bits = store(fmaxf(-most, fminf(low, most)));
  const float scale = half_bits(scale_bits, scale_bf16), offset = offsets ? half_bits(offset_bits, scale_bf16) : -8.f * scale;
  uint32_t word = 0;
  for (int j = 0; j < 8; ++j) {
    float c = scale > 0.f ? rintf((x[j] - offset) / scale) : (offsets ? 0.f : 8.f);
    c = fmaxf(0.f, fminf(c, 15.f));  // (fminf of a NaN is the other operand)
    word |= (first + j < num_dims ? (uint32_t)c : 0u) << (4 * j);
  }
  if (first < (num_dims + 31) / 32 * 32) reinterpret_cast<uint32_t*>(codes + n * ((long long)(num_dims + 31) / 32 * 16))[l] = word;
  if (first % group == 0) {
    const int groups = (num_dims + group - 1) / group;
    scales[n * groups + first / group] = scale_bits;
    if (offsets) offsets[n * groups + first / group] = offset_bits;
  }
}

void launch_pack(const PackArgs& a, hipStream_t stream) {
  if (a.num_rows == 0) return;
  const int lanes = (a.num_dims + a.group - 1) / a.group * (a.group / 8);
  const long long blocks = (a.num_rows * lanes + 255) / 256;
  want(blocks <= 0x7fffffff, "pack: too many rows");
  with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL(pack_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, stream, static_cast<const T*>(a.rows), a.row_stride, a.num_rows,
                       a.num_dims, a.group, lanes, a.codes, static_cast<uint16_t*>(a.scales), static_cast<uint16_t*>(a.offsets),
                       a.scale_type == TYPE_BF16);
  });
  HIP_CHECK(hipGetLastError());
}

// ----------------------------------------------------------------------------------------------- products
struct ScoresArgs {
  const unsigned char* codes;
  const uint16_t *scales, *offsets;
  int scale_bf16;
  long long num_rows;
  int num_dims, group;
  const void* queries;
  long long query_stride;
  int num_queries;
  float alpha;
  const float* bias;
  void* out;
  long long out_stride;
};

template <typename T, typename U>
__global__ void __launch_bounds__(256) scores_kernel(ScoresArgs a) {
  const long long n = (long long)blockIdx.x * 256 + threadIdx.x;
  if (n >= a.num_rows) return;
  const int groups = (a.num_dims + a.group - 1) / a.group;
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(a.codes + n * ((long long)(a.num_dims + 31) / 32 * 16));
  for (int m = blockIdx.y; m < a.num_queries; m += gridDim.y) {
    const T* q = static_cast<const T*>(a.queries) + m * a.query_stride;
    float sum = 0.f;
    for (int g = 0; g < groups; ++g) {
      float dot = 0.f, plain = 0.f;
      for (int k = g * a.group; k < min(a.num_dims, (g + 1) * a.group); ++k) {
        const float x = widen(q[k]);
        const float c = (float)((codes[k >> 3] >> (4 * (k & 7))) & 15u) - (a.offsets ? 0.f : 8.f);
        dot = fmaf(c, x, dot);
        plain += x;
      }
      sum = fmaf(half_bits(a.scales[n * groups + g], a.scale_bf16), dot, sum);
      if (a.offsets) sum = fmaf(half_bits(a.offsets[n * groups + g], a.scale_bf16), plain, sum);
    }
    static_cast<U*>(a.out)[m * a.out_stride + n] = narrow<U>(a.bias ? fmaf(a.alpha, sum, a.bias[n]) : a.alpha * sum);
  }
}

}  // namespace cuhnsw_amd

using namespace cuhnsw_amd;

static void check_packed(long long num_rows, int num_dims, int group, int scale_type) {
  want(num_rows >= 0 && num_dims > 0, "packed rows: bad sizes");
  want(group == 32 || group == 64 || group == 128, "packed rows: the group is 32, 64 or 128 elements");
  want(scale_type == TYPE_F16 || scale_type == TYPE_BF16, "packed rows: scales are float16 or bfloat16");
}

extern "C" {

int cuhnsw_pack_rows(const void* rows, int type, long long row_stride, long long num_rows, int num_dims, int group, void* codes,
                     void* scales, void* offsets, int scale_type, void* stream) {
  return call_guarded([&] {
    check_packed(num_rows, num_dims, group, scale_type);
    want(known_type(type), "pack: unknown element type");
    want(row_stride >= 0, "pack: bad sizes");
    want(num_rows == 0 || (rows && codes && scales), "pack: null argument");
    want((reinterpret_cast<uintptr_t>(codes) & 15) == 0, "pack: codes have to be aligned to 16 bytes");
    launch_pack({rows, type, row_stride, num_rows, num_dims, group, static_cast<unsigned char*>(codes), scales, offsets, scale_type},
                static_cast<hipStream_t>(stream));
  });
}

long long cuhnsw_packed_scores_workspace(long long, int, int, int, int) { return 0; }

int cuhnsw_packed_scores(const void* codes, const void* scales, const void* offsets, int scale_type, long long num_rows, int num_dims,
                         int group, const void* queries, int query_type, long long query_stride, int num_queries, float alpha,
                         const float* bias, void* out, int out_type, long long out_stride, void*, long long, void* stream) {
  return call_guarded([&] {
    check_packed(num_rows, num_dims, group, scale_type);
    want(known_type(query_type) && known_type(out_type), "scores: unknown element type");
    want(num_queries >= 0 && query_stride >= 0 && out_stride >= num_rows, "scores: bad sizes");
    if (num_rows == 0 || num_queries == 0) return;
    want(codes && scales && queries && out, "scores: null argument");
    want((reinterpret_cast<uintptr_t>(codes) & 15) == 0, "scores: codes have to be aligned to 16 bytes");
    want(num_rows <= 0x7fffff00ll, "scores: too many rows");
    const ScoresArgs a{static_cast<const unsigned char*>(codes), static_cast<const uint16_t*>(scales), static_cast<const uint16_t*>(offsets),
                       scale_type == TYPE_BF16, num_rows, num_dims, group, queries, query_stride, num_queries, alpha, bias, out, out_stride};
    with_type(query_type, [&](auto* t) {
      with_type(out_type, [&](auto* u) {
        using T = std::remove_pointer_t<decltype(t)>;
        using U = std::remove_pointer_t<decltype(u)>;
        if constexpr (std::is_same_v<T, U> || std::is_same_v<U, float>)
          hipLaunchKernelGGL((scores_kernel<T, U>), dim3((unsigned)((num_rows + 255) / 256), (unsigned)std::min(num_queries, 65535)), dim3(256), 0,
                             static_cast<hipStream_t>(stream), a);
        else
          throw std::runtime_error("scores: the result has the queries' type or is float32");
      });
    });
    HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
