// The best candidates over the beams of a search and a vocabulary, and the reordering of the beams' states that follows.
//
//   total[b][k][v] = beams[b][k] + x[b][k][v]                                     as the scores are
//   total[b][k][v] = beams[b][k] + x[b][k][v] - log(sum over u of exp(x[b][k][u]))  normalised
//   the `num` largest totals of b over (k, v), largest first; of equal ones the lower k first, then the larger x, then the
//   lower v.
//
// Totals are held in 64 bits: candidates of different beams meet there, and a rounding must not order them.  A NaN counts as
// -infinity, and what is -infinity is never chosen: places that are left over say -infinity, parent -1, token -1.  A finished
// beam has one candidate, the token `end` with the beam's own score.
#include <algorithm>

#include "../../include/cuhnsw_amd.h"
#include "rows.h"

namespace cuhnsw_amd {

constexpr int kMostNum = 256, kMostLists = 4096;

struct SelectArgs {
  const void* scores;
  long long stride_b, stride_k;
  int num_batch, num_beams, num_values;
  const float* beams;            // [num_batch, num_beams] or null
  const unsigned char* finished;  // the same, or null
  int normalise, end, num;
  float* out_totals;
  int *out_parents, *out_tokens;
  double* list_totals;  // per beam: its best min(num, num_values), largest first
  int* list_tokens;
};

// Orders as the values do, +0 and -0 as one; larger keys first means lower places first among equals.
__device__ inline uint64_t order_key(float x, uint32_t place) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~place;
}
__device__ inline float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ inline float score_at(float x) { return fmaxf(x, -INFINITY); }  // (of a NaN: the other operand)

template <typename T>
__global__ void __launch_bounds__(256) select_row_kernel(SelectArgs a) {
  __shared__ uint64_t best[256];
  __shared__ double sums[256];
  const int row = blockIdx.x, b = row / a.num_beams, k = row - b * a.num_beams, tid = threadIdx.x;
  const T* x = static_cast<const T*>(a.scores) + b * a.stride_b + k * a.stride_k;
  const int m = min(a.num, a.num_values);
  const float beam = a.beams ? a.beams[row] : 0.f;
  double* totals = a.list_totals + (long long)row * m;
  int* tokens = a.list_tokens + (long long)row * m;
  if (a.finished && a.finished[row]) {
    for (int i = tid; i < m; i += 256) {
      totals[i] = i == 0 ? (double)beam : -INFINITY;
      tokens[i] = a.end;
    }
    return;
  }
  uint64_t under = ~0ull;
  double top = 0.0, log_sum = 0.0;
  for (int i = 0; i < m; ++i) {
    uint64_t mine = 0;
    for (int v = tid; v < a.num_values; v += 256) {
      const uint64_t key = order_key(score_at(widen(x[v])), (uint32_t)v);
      if (key < under && key > mine) mine = key;
    }
    best[tid] = mine;
    __syncthreads();
    for (int step = 128; step > 0; step >>= 1) {
      if (tid < step && best[tid + step] > best[tid]) best[tid] = best[tid + step];
      __syncthreads();
    }
    under = best[0];
    __syncthreads();
    const float value = key_value(under);
    if (i == 0 && a.normalise) {
      top = value;
      double sum = 0.0;
      for (int v = tid; v < a.num_values; v += 256) {
        const float y = score_at(widen(x[v]));
        sum += y == value ? 1.0 : (double)expf(y - value);
      }
      sums[tid] = sum;
      __syncthreads();
      for (int step = 128; step > 0; step >>= 1) {
        if (tid < step) sums[tid] += sums[tid + step];
        __syncthreads();
      }
      log_sum = log(sums[0]);
    }
    if (tid == 0) {
      double total = value;
      if (a.normalise) total = (value == (float)top ? 0.0 : (double)value - top) - log_sum;
      totals[i] = value == -INFINITY ? -INFINITY : (double)beam + total;
      tokens[i] = (int)~(uint32_t)under;
    }
  }
}

__global__ void __launch_bounds__(64) select_merge_kernel(SelectArgs a) {
  const int b = blockIdx.x, lane = threadIdx.x, m = min(a.num, a.num_values), all = a.num_beams * m;
  const double* totals = a.list_totals + (long long)b * all;
  const int* tokens = a.list_tokens + (long long)b * all;
  double last = INFINITY;
  int last_at = -1;
  for (int i = 0; i < a.num; ++i) {
    double best = -INFINITY;
    int at = all;
    for (int c = lane; c < all; c += 64) {
      const double t = totals[c];
      const bool left = t < last || (t == last && c > last_at);
      if (left && t > best) best = t, at = c;
    }
    for (int step = 1; step < 64; step <<= 1) {
      const double t = __shfl_xor(best, step);
      const int c = __shfl_xor(at, step);
      if (t > best || (t == best && c < at)) best = t, at = c;
    }
    const bool there = best > -INFINITY;
    if (lane == 0) {
      a.out_totals[(long long)b * a.num + i] = (float)best;
      a.out_parents[(long long)b * a.num + i] = there ? at / m : -1;
      a.out_tokens[(long long)b * a.num + i] = there ? tokens[at] : -1;
    }
    last = best;
    last_at = at;
  }
}

// ----------------------------------------------------------------------------------------------- states
constexpr int kMostStates = 32;
struct ReorderArgs {
  const unsigned char* from[kMostStates];
  unsigned char* to[kMostStates];
  long long stride_b[kMostStates], stride_k[kMostStates], bytes[kMostStates];  // in bytes; the results are dense
  const int* parents;
  long long parent_stride_b, parent_stride_k;
  int num_beams, num_picked;
};

__global__ void __launch_bounds__(256) reorder_kernel(ReorderArgs a) {
  const int s = blockIdx.z, row = blockIdx.y, b = row / a.num_picked, j = row - b * a.num_picked;
  const int parent = a.parents[b * a.parent_stride_b + j * a.parent_stride_k];
  const bool there = parent >= 0 && parent < a.num_beams;
  const unsigned char* from = a.from[s] + b * a.stride_b[s] + (there ? parent : 0) * a.stride_k[s];
  unsigned char* to = a.to[s] + row * a.bytes[s];
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < a.bytes[s]; i += (long long)gridDim.x * 256) to[i] = there ? from[i] : 0;
}

struct SelectScratch {
  double* totals;
  int* tokens;
  size_t bytes;
  SelectScratch(void* memory, long long rows, int num) {
    WorkspaceParts s(memory);
    totals = s.part<double>((size_t)rows * num);
    tokens = s.part<int>((size_t)rows * num);
    bytes = s.used();
  }
};

}  // namespace cuhnsw_amd

using namespace cuhnsw_amd;

extern "C" {

long long cuhnsw_select_beams_workspace(int num_batch, int num_beams, int num_values, int num) {
  if (num_batch <= 0 || num_beams <= 0 || num_values <= 0 || num <= 0) return 0;
  return (long long)SelectScratch(nullptr, (long long)num_batch * num_beams, std::min(num, num_values)).bytes;
}

int cuhnsw_select_beams(const void* scores, int type, long long stride_b, long long stride_k, int num_batch, int num_beams, int num_values,
                        const float* beams, const unsigned char* finished, int end, int normalise, int num, float* out_totals,
                        int* out_parents, int* out_tokens, void* workspace, long long workspace_bytes, void* stream) {
  return call_guarded([&] {
    want(known_type(type), "select: unknown element type");
    want(num_batch >= 0 && num_beams > 0 && num_values > 0, "select: bad sizes");
    want(num > 0 && num <= kMostNum, "select: between 1 and 256 candidates can be asked for");
    want((long long)num_beams * std::min(num, num_values) <= kMostLists, "select: more than 4096 candidates of all beams (beams times candidates asked for)");
    want((long long)num_batch * num_beams <= 0x7fffffff, "select: too many rows");
    if (num_batch == 0) return;
    want(scores && out_totals && out_parents && out_tokens, "select: null argument");
    want(!finished || (end >= 0 && end < num_values), "select: the token that ends a sequence is outside the vocabulary");
    const SelectScratch w(workspace, (long long)num_batch * num_beams, std::min(num, num_values));
    want(workspace && workspace_bytes >= (long long)w.bytes, "select: the workspace is too small");
    const SelectArgs a{scores, stride_b, stride_k, num_batch, num_beams, num_values, beams, finished, normalise, end, num,
                       out_totals, out_parents, out_tokens, w.totals, w.tokens};
    hipStream_t s = static_cast<hipStream_t>(stream);
    with_type(type, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      hipLaunchKernelGGL(select_row_kernel<T>, dim3((unsigned)(num_batch * num_beams)), dim3(256), 0, s, a);
    });
    hipLaunchKernelGGL(select_merge_kernel, dim3((unsigned)num_batch), dim3(64), 0, s, a);
    HIP_CHECK(hipGetLastError());
  });
}

int cuhnsw_reorder_states(const void* const* from, void* const* to, const long long* stride_b, const long long* stride_k,
                          const long long* bytes, int num_states, const int* parents, long long parent_stride_b,
                          long long parent_stride_k, int num_batch, int num_beams, int num_picked, void* stream) {
  return call_guarded([&] {
    want(num_states >= 0 && num_batch >= 0 && num_beams > 0 && num_picked >= 0, "reorder: bad sizes");
    if (num_states == 0 || num_batch == 0 || num_picked == 0) return;
    want(from && to && stride_b && stride_k && bytes && parents, "reorder: null argument");
    want((long long)num_batch * num_picked <= 65535, "reorder: more than 65535 rows");
    for (int first = 0; first < num_states; first += kMostStates) {
      ReorderArgs a{};
      const int count = std::min(kMostStates, num_states - first);
      long long most = 0;
      for (int i = 0; i < count; ++i) {
        a.from[i] = static_cast<const unsigned char*>(from[first + i]);
        a.to[i] = static_cast<unsigned char*>(to[first + i]);
        a.stride_b[i] = stride_b[first + i];
        a.stride_k[i] = stride_k[first + i];
        a.bytes[i] = bytes[first + i];
        want(a.bytes[i] >= 0 && (a.bytes[i] == 0 || (a.from[i] && a.to[i])), "reorder: null argument");
        most = std::max(most, a.bytes[i]);
      }
      if (most == 0) continue;
      a.parents = parents;
      a.parent_stride_b = parent_stride_b;
      a.parent_stride_k = parent_stride_k;
      a.num_beams = num_beams;
      a.num_picked = num_picked;
      hipLaunchKernelGGL(reorder_kernel, dim3((unsigned)std::min<long long>((most + 255) / 256, 1024), (unsigned)(num_batch * num_picked), (unsigned)count),
                         dim3(256), 0, static_cast<hipStream_t>(stream), a);
      HIP_CHECK(hipGetLastError());
    }
  });
}

}  // extern "C"
