// Rows of a table by id, and the gradient of that.
//
//   out[t] = scale * table[ids[t]]                         (zeros where ids[t] is outside [0, num_rows))
//   grad[v] = scale * sum over t with ids[t] = v of g[t]   (t ascending; zeros for rows that no id names)
//
// Products and sums are held in 32 bits and rounded once, to nearest, when they are stored.
#include <algorithm>

#include "../../include/cuhnsw_amd.h"
#include "rows.h"

namespace cuhnsw_amd {

__device__ inline long long id_at(const void* ids, int ids_64, long long t) {
  return ids_64 ? reinterpret_cast<const long long*>(ids)[t] : (long long)reinterpret_cast<const int*>(ids)[t];
}

// ---------------------------------------------------------------------------------------------- lookup
template <typename T, typename U>
__global__ void __launch_bounds__(256) lookup_kernel(const T* table, long long num_rows, long long row_stride, int num_dims,
                                                     const void* ids, int ids_64, long long num_ids, float scale, U* out) {
  const long long total = num_ids * num_dims;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long t = i / num_dims, d = i - t * num_dims, id = id_at(ids, ids_64, t);
    out[i] = narrow<U>(id >= 0 && id < num_rows ? scale * widen(table[id * row_stride + d]) : 0.f);
  }
}

void launch_lookup(const LookupArgs& a, hipStream_t stream) {
  if (a.num_ids == 0) return;
  const long long blocks = std::min<long long>((a.num_ids * a.num_dims + 255) / 256, 1 << 16);
  with_type(a.table_type, [&](auto* t) {
    with_type(a.out_type, [&](auto* u) {
      using T = std::remove_pointer_t<decltype(t)>;
      using U = std::remove_pointer_t<decltype(u)>;
      if constexpr (std::is_same_v<T, U> || std::is_same_v<U, float>) {
        hipLaunchKernelGGL((lookup_kernel<T, U>), dim3((unsigned)blocks), dim3(256), 0, stream, static_cast<const T*>(a.table), a.num_rows,
                           a.row_stride, a.num_dims, a.ids, a.ids_64, a.num_ids, a.scale, static_cast<U*>(a.out));
      } else {
        throw std::runtime_error("lookup: the result has the table's type or is float32");
      }
    });
  });
  HIP_CHECK(hipGetLastError());
}

// ------------------------------------------------------------------------------------ ids in order
// A stable sort of (id, place) by id, least significant digit first: places of one id stay in ascending order, so the sums do
// not depend on how the work was spread.  Ids outside the table take the key num_rows, behind all others.  One pass is two
// launches: every workgroup counts the digits of its stretch of ids; then each adds up the counts of the others before it,
// ranks its own ids by ballots among the lanes that hold the same digit, and sends them to their places.
constexpr int kSortThreads = 256, kSortWaves = 4, kSortBlocks = 128, kMostDigits = 2048;

struct SortPlan {
  int passes, bits;   // digits of `bits` bits
  int blocks, chunk;  // stretches of `chunk` ids (a multiple of kSortThreads)
};
static SortPlan sort_plan(long long num_ids, long long num_rows) {
  int bits = 1;
  while ((1ll << bits) <= num_rows) ++bits;
  SortPlan p;
  p.passes = (bits + 10) / 11;
  p.bits = (bits + p.passes - 1) / p.passes;
  const long long rounds = std::max<long long>(4, (num_ids + (long long)kSortBlocks * kSortThreads - 1) / ((long long)kSortBlocks * kSortThreads));
  p.chunk = (int)(rounds * kSortThreads);
  p.blocks = (int)((num_ids + p.chunk - 1) / p.chunk);
  return p;
}

struct SortInput {  // the ids themselves in the first pass, (key, place) pairs afterwards
  const void* ids;
  int ids_64;
  int num_rows;
  const int* keys;
  const int* places;
};
__device__ inline int sort_key(const SortInput& in, int i) {
  if (in.keys) return in.keys[i];
  const long long id = id_at(in.ids, in.ids_64, i);
  return id >= 0 && id < in.num_rows ? (int)id : in.num_rows;
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortInput in, int num_ids, int chunk, int shift, int digits, int* counts) {
  __shared__ int count[kMostDigits];
  for (int d = threadIdx.x; d < digits; d += kSortThreads) count[d] = 0;
  __syncthreads();
  const int begin = blockIdx.x * chunk, end = min(num_ids, begin + chunk);
  for (int i = begin + threadIdx.x; i < end; i += kSortThreads) atomicAdd(&count[(sort_key(in, i) >> shift) & (digits - 1)], 1);
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) counts[blockIdx.x * digits + d] = count[d];
}

__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(SortInput in, int num_ids, int chunk, int shift, int digits, int bits,
                                                                  const int* counts, int* keys, int* places) {
  __shared__ int next[kMostDigits];               // where the next id with a digit goes
  __shared__ int wave_count[kSortWaves][kMostDigits];
  __shared__ int wave_sum[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // ids with a smaller digit anywhere, and with the same digit in an earlier stretch; each thread has consecutive digits
  const int per_thread = (digits + kSortThreads - 1) / kSortThreads;
  int mine = 0;
  for (int j = 0; j < per_thread; ++j) {
    const int d = tid * per_thread + j;
    if (d >= digits) break;
    int before = 0, all = 0;
    for (int b = 0; b < (int)gridDim.x; ++b) {
      const int n = counts[b * digits + d];
      before += b < (int)blockIdx.x ? n : 0;
      all += n;
    }
    next[d] = before + mine;
    mine += all;
  }
  int upto = mine;
  for (int step = 1; step < 64; step <<= 1) {
    const int other = __shfl_up(upto, step);
    if (lane >= step) upto += other;
  }
  if (lane == 63) wave_sum[wave] = upto;
  __syncthreads();
  int base = upto - mine;
  for (int w = 0; w < wave; ++w) base += wave_sum[w];
  for (int j = 0; j < per_thread; ++j) {
    const int d = tid * per_thread + j;
    if (d < digits) next[d] += base;
  }
  const int begin = blockIdx.x * chunk, end = min(num_ids, begin + chunk);
  for (int start = begin; start < end; start += kSortThreads) {  // (the same number of rounds for every wavefront)
    for (int d = tid; d < digits; d += kSortThreads)
      for (int w = 0; w < kSortWaves; ++w) wave_count[w][d] = 0;
    __syncthreads();
    const int i = start + tid;
    const bool there = i < end;
    const int key = there ? sort_key(in, i) : 0;
    const int d = (key >> shift) & (digits - 1);
    unsigned long long peers = __ballot(there);
    for (int b = 0; b < bits; ++b) {
      const unsigned long long with = __ballot((d >> b) & 1);
      peers &= (d >> b) & 1 ? with : ~with;
    }
    const int rank = __popcll(peers & ((1ull << lane) - 1));
    if (there && rank == 0) wave_count[wave][d] = __popcll(peers);
    __syncthreads();
    if (there) {
      int at = next[d] + rank;
      for (int w = 0; w < wave; ++w) at += wave_count[w][d];
      keys[at] = key;
      places[at] = in.keys ? in.places[i] : i;
    }
    __syncthreads();
    for (int x = tid; x < digits; x += kSortThreads)
      for (int w = 0; w < kSortWaves; ++w) next[x] += wave_count[w][x];
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------- gradient
// first place in [0, n) whose key is at least `key`
__device__ inline int lower_bound(const int* keys, int n, int key) {
  int low = 0, high = n;
  while (low < high) {
    const int mid = (low + high) >> 1;
    if (keys[mid] < key) low = mid + 1;
    else high = mid;
  }
  return low;
}

template <typename T, typename U>
__global__ void __launch_bounds__(256) grad_kernel(const T* grad, long long grad_stride, const int* keys, const int* places, int num_ids,
                                                   int num_rows, int num_dims, float scale, U* out) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= num_rows) return;
  const int begin = lower_bound(keys, num_ids, row), end = lower_bound(keys, num_ids, row + 1);
  for (int d = lane; d < num_dims; d += 64) {
    float sum = 0.f;
    for (int i = begin; i < end; ++i) sum += widen(grad[(long long)places[i] * grad_stride + d]);
    out[(long long)row * num_dims + d] = narrow<U>(scale * sum);
  }
}

struct GradScratch {
  int *keys[2], *places[2], *counts;
  size_t bytes;
  GradScratch(void* memory, long long num_ids, const SortPlan& p) {
    WorkspaceParts s(memory);
    for (int i = 0; i < 2; ++i) {
      keys[i] = s.part<int>((size_t)num_ids);
      places[i] = s.part<int>((size_t)num_ids);
    }
    counts = s.part<int>((size_t)p.blocks << p.bits);
    bytes = s.used();
  }
};

}  // namespace cuhnsw_amd

using namespace cuhnsw_amd;

extern "C" {

int cuhnsw_lookup_rows(const void* table, int table_type, long long num_rows, long long row_stride, int num_dims, const void* ids,
                       int ids_64, long long num_ids, float scale, void* out, int out_type, void* stream) {
  return call_guarded([&] {
    want(known_type(table_type) && known_type(out_type), "lookup: unknown element type");
    want(num_rows >= 0 && num_dims > 0 && num_ids >= 0 && row_stride >= 0, "lookup: bad sizes");
    want(num_ids == 0 || (ids && out && (table || num_rows == 0)), "lookup: null argument");
    launch_lookup({table, table_type, num_rows, row_stride, num_dims, ids, ids_64, num_ids, scale, out, out_type},
                  static_cast<hipStream_t>(stream));
  });
}

long long cuhnsw_lookup_grad_workspace(long long num_ids, long long num_rows, int num_dims) {
  if (num_ids <= 0 || num_rows <= 0 || num_dims <= 0) return 0;
  return (long long)GradScratch(nullptr, num_ids, sort_plan(num_ids, num_rows)).bytes;
}

int cuhnsw_lookup_rows_grad(const void* grad, int grad_type, long long grad_stride, const void* ids, int ids_64, long long num_ids,
                            long long num_rows, int num_dims, float scale, void* out, int out_type, void* workspace,
                            long long workspace_bytes, void* stream) {
  return call_guarded([&] {
    want(known_type(grad_type) && known_type(out_type), "lookup gradient: unknown element type");
    want(num_rows >= 0 && num_dims > 0 && num_ids >= 0 && grad_stride >= 0, "lookup gradient: bad sizes");
    want(num_ids <= 1 << 30 && num_rows < 0x7fffffff, "lookup gradient: more than 2^30 ids or 2^31 - 2 rows");
    want(num_rows == 0 || out, "lookup gradient: null argument");
    want(num_ids == 0 || (grad && ids), "lookup gradient: null argument");
    if (num_rows == 0) return;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int *keys = nullptr, *places = nullptr;
    if (num_ids > 0) {
      const SortPlan p = sort_plan(num_ids, num_rows);
      const GradScratch w(workspace, num_ids, p);
      want(workspace && workspace_bytes >= (long long)w.bytes, "lookup gradient: the workspace is too small");
      for (int pass = 0; pass < p.passes; ++pass) {
        const SortInput in{ids, ids_64, (int)num_rows, pass ? w.keys[(pass - 1) & 1] : nullptr, pass ? w.places[(pass - 1) & 1] : nullptr};
        hipLaunchKernelGGL(sort_count_kernel, dim3(p.blocks), dim3(kSortThreads), 0, s, in, (int)num_ids, p.chunk, pass * p.bits, 1 << p.bits,
                           w.counts);
        hipLaunchKernelGGL(sort_place_kernel, dim3(p.blocks), dim3(kSortThreads), 0, s, in, (int)num_ids, p.chunk, pass * p.bits, 1 << p.bits,
                           p.bits, w.counts, w.keys[pass & 1], w.places[pass & 1]);
      }
      keys = w.keys[(p.passes - 1) & 1];
      places = w.places[(p.passes - 1) & 1];
    }
    with_type(grad_type, [&](auto* t) {
      with_type(out_type, [&](auto* u) {
        using T = std::remove_pointer_t<decltype(t)>;
        using U = std::remove_pointer_t<decltype(u)>;
        if constexpr (std::is_same_v<T, U> || std::is_same_v<T, float>) {
          hipLaunchKernelGGL((grad_kernel<T, U>), dim3((unsigned)((num_rows + 3) / 4)), dim3(256), 0, s, static_cast<const T*>(grad), grad_stride,
                             keys, places, (int)num_ids, (int)num_rows, num_dims, scale, static_cast<U*>(out));
        } else {
          throw std::runtime_error("lookup gradient: the gradient has the table's type or is float32");
        }
      });
    });
    HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
