// Rows of a table by id, and the gradient of that.
//
//   out[t] = scale * table[ids[t]]                         (zeros where ids[t] is outside [0, num_rows))
//   grad[v] = scale * sum over t with ids[t] = v of g[t]   (zeros for rows that no id names; in which order is fixed by sizes and ids)
//
// Products and sums are held in 32 bits and rounded once, to nearest, when they are stored.
#include <algorithm>

#include "../../include/cuhnsw_amd.h"
#include "rows.h"

namespace cuhnsw_amd {

__device__ inline long long id_at(const void* ids, int ids_64, long long t) {
  return ids_64 ? reinterpret_cast<const long long*>(ids)[t] : (long long)reinterpret_cast<const int*>(ids)[t];
}

// A row in whole vectors of VE elements: the last one begins VE before the end, and where that overlaps the one before it both
// hold the same.  (Global memory takes 16 bytes from and to any address that fits an element, so rows of any length and
// stride move 16 bytes at a time; rows of fewer elements than a vector go one by one.)
template <int VE>
__device__ __host__ inline int vectors_of(int num_dims) {
  return (num_dims + VE - 1) / VE;
}
template <int VE>
__device__ inline int vector_at(int v, int num_dims) {
  return min(v * VE, num_dims - VE);
}
// A large result goes past the caches, whose lines would otherwise all be written back when the kernel ends: 50 003 rows of 960
// float16 (96 MB) in 38.5 us instead of 44, 131 072 x 1024 bfloat16 of a gradient 6 us sooner.
constexpr long long kStreamedFrom = 64ll << 20;
template <bool STREAMED, typename U, int VE>
__device__ inline void store_result(U* to, const LoosePack<U, VE>& p) {
  if constexpr (STREAMED && sizeof(p) == 16) {
    typedef uint32_t vector_t __attribute__((ext_vector_type(4)));
    typedef uint32_t loose_t __attribute__((ext_vector_type(4), aligned(2)));
    __builtin_nontemporal_store(__builtin_bit_cast(vector_t, p), reinterpret_cast<loose_t*>(to));
  } else {
    *reinterpret_cast<LoosePack<U, VE>*>(to) = p;
  }
}
template <typename F>
void with_flag(bool flag, F&& f) {
  if (flag) f(std::true_type());
  else f(std::false_type());
}
// lanes that share a row: the power of two that its vectors fill at least half of, a wavefront at most
inline int lanes_of(int vectors) {
  int lanes = 1;
  while (lanes < vectors && lanes < 64) lanes <<= 1;
  return lanes;
}
// f with the elements of a vector as a constant
template <typename T, typename F>
void with_vector(int num_dims, F&& f) {
  constexpr int VE = 16 / sizeof(T);
  if (num_dims >= VE) f(std::integral_constant<int, VE>());
  else f(std::integral_constant<int, 1>());
}

// ---------------------------------------------------------------------------------------------- lookup
// Bound by memory: each row is fetched once and written once, four rows of a lane's in flight (from 2048 workgroups on, below that there
// are too few rows for four each).  50 003 of 400 000 rows of 960 float16: 192 MB in 37.5 us, 5.1 TB/s (a copy of as much takes 39 us,
// 5.2 TB/s); 65 536 tokens of 1024 bfloat16 46 us.  A few rows take a launch: 3 us.
template <typename T, typename U, int VE, bool STREAMED>
__global__ void __launch_bounds__(256) lookup_kernel(const T* table, long long num_rows, long long row_stride, int num_dims,
                                                     const void* ids, int ids_64, long long num_ids, float scale, U* out, int lanes) {
  constexpr int kAtOnce = 4;
  const int vectors = vectors_of<VE>(num_dims), lane = threadIdx.x & (lanes - 1);
  const long long groups = (long long)gridDim.x * (256 / lanes);
  for (long long t0 = (long long)blockIdx.x * (256 / lanes) + threadIdx.x / lanes; t0 < num_ids; t0 += kAtOnce * groups) {
    const T* from[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const long long t = t0 + j * groups, id = t < num_ids ? id_at(ids, ids_64, t) : -1;
      from[j] = id >= 0 && id < num_rows ? table + id * row_stride : nullptr;
    }
    for (int v = lane; v < vectors; v += lanes) {
      const int d = vector_at<VE>(v, num_dims);
      LoosePack<T, VE> x[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (from[j]) x[j] = *reinterpret_cast<const LoosePack<T, VE>*>(from[j] + d);
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const long long t = t0 + j * groups;
        if (t >= num_ids) break;
        LoosePack<U, VE> y;
#pragma unroll
        for (int e = 0; e < VE; ++e) y.at[e] = narrow<U>(from[j] ? scale * widen(x[j].at[e]) : 0.f);
        store_result<STREAMED>(out + t * num_dims + d, y);
      }
    }
  }
}

void launch_lookup(const LookupArgs& a, hipStream_t stream) {
  if (a.num_ids == 0) return;
  with_type(a.table_type, [&](auto* t) {
    with_type(a.out_type, [&](auto* u) {
      using T = std::remove_pointer_t<decltype(t)>;
      using U = std::remove_pointer_t<decltype(u)>;
      if constexpr (std::is_same_v<T, U> || std::is_same_v<U, float>) {
        with_vector<T>(a.num_dims, [&](auto ve) {
          constexpr int VE = decltype(ve)::value;
          const int lanes = lanes_of(vectors_of<VE>(a.num_dims)), groups = 256 / lanes;
          const long long blocks = std::min<long long>((a.num_ids + groups - 1) / groups, 1 << 20);
          with_flag(a.num_ids * a.num_dims * (long long)sizeof(U) >= kStreamedFrom, [&](auto streamed) {
            hipLaunchKernelGGL((lookup_kernel<T, U, VE, decltype(streamed)::value>), dim3((unsigned)(blocks <= 2048 ? blocks : (blocks + 3) / 4)),
                               dim3(256), 0, stream, static_cast<const T*>(a.table), a.num_rows, a.row_stride, a.num_dims, a.ids, a.ids_64,
                               a.num_ids, a.scale, static_cast<U*>(a.out), lanes);
          });
        });
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
// and each of its wavefronts ranks a quarter of the stretch by ballots among the lanes that hold the same digit.  65 536 ids of
// 17 bits: twice 4.8 + 12.2 us, all of it waits; with stretches of 512 or 2048 ids instead of 1024 the second launch takes
// 13.8 and 14.3.
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
  __shared__ int next[kSortWaves][kMostDigits];  // first how many ids a wavefront has with a digit, then where its next one goes
  __shared__ int wave_sum[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int d = tid; d < digits; d += kSortThreads)
    for (int w = 0; w < kSortWaves; ++w) next[w][d] = 0;
  __syncthreads();
  const int quarter = chunk / kSortWaves, begin = blockIdx.x * chunk + wave * quarter, end = min(num_ids, begin + quarter);
  for (int i = begin + lane; i < end; i += 64) atomicAdd(&next[wave][(sort_key(in, i) >> shift) & (digits - 1)], 1);
  // ids with a smaller digit anywhere, and with the same digit in an earlier stretch; each thread has consecutive digits
  constexpr int kDigits = kMostDigits / kSortThreads;
  const int per_thread = (digits + kSortThreads - 1) / kSortThreads;
  int before[kDigits], mine = 0;
#pragma unroll
  for (int j = 0; j < kDigits; ++j) {
    const int d = tid * per_thread + j;
    before[j] = 0;
    if (j >= per_thread || d >= digits) continue;
    int all = 0;
#pragma unroll 32
    for (int b = 0; b < (int)gridDim.x; ++b) {
      const int n = counts[b * digits + d];
      before[j] += b < (int)blockIdx.x ? n : 0;
      all += n;
    }
    before[j] += mine;
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
#pragma unroll
  for (int j = 0; j < kDigits; ++j) {
    const int d = tid * per_thread + j;
    if (j >= per_thread || d >= digits) continue;
    int at = base + before[j];
    for (int w = 0; w < kSortWaves; ++w) {
      const int n = next[w][d];
      next[w][d] = at;
      at += n;
    }
  }
  __syncthreads();
  for (int i = begin + lane; i - lane < end; i += 64) {
    const bool there = i < end;
    const int key = there ? sort_key(in, i) : 0, d = (key >> shift) & (digits - 1);
    unsigned long long peers = __ballot(there);
    for (int b = 0; b < bits; ++b) {
      const unsigned long long with = __ballot((d >> b) & 1);
      peers &= (d >> b) & 1 ? with : ~with;
    }
    const int rank = __popcll(peers & ((1ull << lane) - 1));
    int at = 0;
    if (there && rank == 0) at = atomicAdd(&next[wave][d], __popcll(peers));
    at = __shfl(at, there ? __ffsll((long long)peers) - 1 : 0) + rank;
    if (there) {
      keys[at] = key;
      places[at] = in.keys ? in.places[i] : i;
    }
  }
}

// ------------------------------------------------------------------------------------------- gradient
// A workgroup has a stretch of rows and the (key, place) pairs of theirs, in order: out of the sorted list, or, where there
// are few ids (up to kFew), picked out of all of them and sorted in LDS: one launch instead of six.  A row of up to kTogether places
// is a group of lanes' own; the places of a longer one are divided among all groups of the workgroup.  In the sorted list
// stretches of kLong places of one id have been summed before (grad_long_kernel), so that no row is much longer
// than that.  Which sum is formed in which order depends on sizes and ids alone.
//
// Times in us.  Few against sorted, skewed ids: 100 000 x 50 fp32, 64 ids 6.8 and 19.0, 1000 ids 13.4 and 31.4, 2000 ids 24.1 and
// 36.7; 131 072 x 1024 bf16, 2000 ids 49.1 and 74.6, 4000 ids 90.7 and 82.6.  65 536 ids of a skewed vocabulary into 131 072 x 1024
// bf16: 178 with the places of rows longer than kTogether divided, 676 without.
constexpr int kLong = 64, kTogether = 16, kFew = 2048, kMostRows = 128;

// sum of the vectors of the items [from, to), in order, up to eight of them in flight; where(i): item i's address
template <typename T, int VE, int N, typename F>
__device__ inline void add_items(int from, int count, F&& where, float (&sum)[VE]) {
  LoosePack<T, VE> x[N];
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (j < count) x[j] = *where(from + j);
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (j < count)
#pragma unroll
      for (int e = 0; e < VE; ++e) sum[e] += widen(x[j].at[e]);
}
template <typename T, int VE, typename F>
__device__ inline void sum_items(int from, int to, F&& where, float (&sum)[VE]) {
#pragma unroll
  for (int e = 0; e < VE; ++e) sum[e] = 0.f;
  int i = from;
  for (; i + 8 <= to; i += 8) add_items<T, VE, 8>(i, 8, where, sum);
  if (i + 4 <= to) {
    add_items<T, VE, 4>(i, 4, where, sum);
    i += 4;
  }
  if (i < to) add_items<T, VE, 3>(i, to - i, where, sum);
}

// The same by the whole workgroup, a contiguous part of the items for every group of lanes; the first group adds the parts to
// what it has.  parts: 256 x VE places in LDS.
template <typename T, int VE, typename F>
__device__ inline void sum_items_together(int items, int lanes, F&& where, float (&sum)[VE], float* parts) {
  const int groups = 256 / lanes, group = threadIdx.x / lanes, share = (items + groups - 1) / groups;
  float mine[VE];
  sum_items<T, VE>(min(items, group * share), min(items, (group + 1) * share), where, mine);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < VE; ++e) parts[threadIdx.x * VE + e] = mine[e];
  __syncthreads();
  if (group == 0)
    for (int g = 0; g < min(groups, items); ++g)
#pragma unroll
      for (int e = 0; e < VE; ++e) sum[e] += parts[(g * lanes + threadIdx.x) * VE + e];
}

template <bool STREAMED, typename U, int VE>
__device__ inline void store(U* to, const float (&x)[VE], float scale) {
  LoosePack<U, VE> p;
#pragma unroll
  for (int e = 0; e < VE; ++e) p.at[e] = narrow<U>(scale * x[e]);
  store_result<STREAMED>(to, p);
}

struct GradArgs {
  const void* grad;
  long long grad_stride;
  const void* ids;  // few ids: themselves
  int ids_64;
  const int *keys, *places;  // many: in order
  float* long_sums;          // [num_ids / kLong, num_dims]: sums of the stretches that are one id's alone
  int* bounds;               // where every workgroup's rows begin in the sorted list, and the end of the last one's
  int num_stretches, num_blocks;
  int num_ids, num_rows, num_dims;
  float scale;
  void* out;
  int lanes, rows;  // lanes that share a row, rows of a workgroup
  int first_block;  // of this launch
};
// A launch has fewer than 2^32 threads: what more workgroups have to do goes in several.
constexpr long long kMostBlocks = 0xffffff;
template <typename F>
void in_launches(GradArgs& g, long long blocks, F&& launch) {
  for (long long first = 0; first < blocks; first += kMostBlocks) {
    g.first_block = (int)first;
    launch(dim3((unsigned)std::min(kMostBlocks, blocks - first)));
    HIP_CHECK(hipGetLastError());  // (what comes next reads what this one writes)
  }
}

// Stretches of the sorted list that are one id's alone; and, by the workgroups behind those, where the rows of grad_kernel's
// workgroups begin: a search for each thread, which would be every one's first wait there.
template <typename T, int VE>
__global__ void __launch_bounds__(256) grad_long_kernel(GradArgs a) {
  __shared__ float parts[256 * VE];
  const int block = a.first_block + blockIdx.x;
  if (block >= a.num_stretches) {
    const int i = (block - a.num_stretches) * 256 + threadIdx.x;
    if (i > a.num_blocks) return;
    const int row = (int)min((long long)i * a.rows, (long long)a.num_rows);
    int low = 0, high = a.num_ids;
    while (low < high) {
      const int mid = (low + high) >> 1;
      if (a.keys[mid] < row) low = mid + 1;
      else high = mid;
    }
    a.bounds[i] = low;
    return;
  }
  const int first = block * kLong, key = a.keys[first];
  if (key >= a.num_rows || a.keys[first + kLong - 1] != key) return;
  const int lane = threadIdx.x & (a.lanes - 1), vectors = vectors_of<VE>(a.num_dims);
  const T* grad = static_cast<const T*>(a.grad);
  for (int v0 = 0; v0 < vectors; v0 += a.lanes) {
    const int d = vector_at<VE>(min(v0 + lane, vectors - 1), a.num_dims);
    float sum[VE] = {};
    sum_items_together<T, VE>(kLong, a.lanes, [&](int i) {
      return reinterpret_cast<const LoosePack<T, VE>*>(grad + (long long)a.places[first + i] * a.grad_stride + d);
    }, sum, parts);
    if (threadIdx.x < a.lanes) store<false>(a.long_sums + (long long)block * a.num_dims + d, sum, 1.f);
  }
}

template <typename T, typename U, int VE, bool FEW, bool STREAMED>
__global__ void __launch_bounds__(256) grad_kernel(GradArgs a) {
  __shared__ int first[kMostRows], last[kMostRows];
  __shared__ int long_rows[kMostRows], long_count;
  __shared__ int picked_count;
  __shared__ float parts[256 * VE];
  extern __shared__ uint64_t picked[];  // few ids: [num_ids], and their places in order behind them
  int* in_order = reinterpret_cast<int*>(picked + (FEW ? a.num_ids : 0));
  const int tid = threadIdx.x, block = a.first_block + blockIdx.x, row0 = block * a.rows, rows = min(a.rows, a.num_rows - row0);
  for (int r = tid; r < rows; r += 256) first[r] = last[r] = 0;
  if (tid == 0) long_count = 0;
  if (FEW) {
    if (tid == 0) picked_count = 0;
    __syncthreads();
    for (int i = tid; i < a.num_ids; i += 256) {
      const long long r = id_at(a.ids, a.ids_64, i) - row0;
      if (r >= 0 && r < rows) picked[atomicAdd(&picked_count, 1)] = (uint64_t)r << 32 | (uint32_t)i;
    }
    __syncthreads();
    const int count = picked_count;
    if (count <= 256) {
      if (tid < count) {
        const uint64_t mine = picked[tid];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += picked[j] < mine;
        in_order[rank] = tid;
      }
    } else {  // (the keys of many change places themselves)
      int size = 512;
      while (size < count) size <<= 1;
      for (int run = 2; run <= size; run <<= 1)
        for (int step = run >> 1; step > 0; step >>= 1) {
          __syncthreads();
          for (int i = tid; i < size / 2; i += 256) {
            // (always rising, so that what is behind the last one can be left out: the first step of a run compares mirrored places)
            const int in_step = i & (step - 1), low = (i - in_step) * 2;
            const int x = low + in_step, y = step == run >> 1 ? low + 2 * step - 1 - in_step : x + step;
            if (y < count && picked[y] < picked[x]) {
              const uint64_t swapped = picked[x];
              picked[x] = picked[y];
              picked[y] = swapped;
            }
          }
        }
      __syncthreads();
      for (int i = tid; i < count; i += 256) in_order[i] = i;
    }
    __syncthreads();
    for (int i = tid; i < count; i += 256) {
      const uint64_t mine = picked[in_order[i]];
      const int r = (int)(mine >> 32);
      if (i == 0 || (int)(picked[in_order[i - 1]] >> 32) != r) first[r] = i;
      if (i + 1 == count || (int)(picked[in_order[i + 1]] >> 32) != r) last[r] = i + 1;
    }
    __syncthreads();
    for (int i = tid; i < count; i += 256) in_order[i] = (int)(uint32_t)picked[in_order[i]];
  } else {
    const int begin = a.bounds[block], end = a.bounds[block + 1];
    __syncthreads();
    for (int i = begin + tid; i < end; i += 256) {
      const int key = a.keys[i];
      if (i == begin || a.keys[i - 1] != key) first[key - row0] = i;
      if (i + 1 == end || a.keys[i + 1] != key) last[key - row0] = i + 1;
    }
  }
  __syncthreads();
  const T* grad = static_cast<const T*>(a.grad);
  U* out = static_cast<U*>(a.out) + (long long)row0 * a.num_dims;
  const int lane = tid & (a.lanes - 1), groups = 256 / a.lanes, vectors = vectors_of<VE>(a.num_dims);
  for (int r = tid / a.lanes; r < rows; r += groups) {
    const int from = first[r], to = last[r];
    if (to - from > kTogether) {
      if (lane == 0) long_rows[atomicAdd(&long_count, 1)] = r;
      continue;
    }
    for (int v = lane; v < vectors; v += a.lanes) {
      const int d = vector_at<VE>(v, a.num_dims);
      float sum[VE];
      sum_items<T, VE>(from, to, [&](int i) {
        return reinterpret_cast<const LoosePack<T, VE>*>(grad + (long long)(FEW ? in_order[i] : a.places[i]) * a.grad_stride + d);
      }, sum);
      store<STREAMED>(out + (long long)r * a.num_dims + d, sum, a.scale);
    }
  }
  __syncthreads();
  for (int l = 0; l < long_count; ++l) {
    const int r = long_rows[l], from = first[r], to = last[r];
    // its places up to the first whole stretch, the whole stretches, the places behind them
    const int whole = (from + kLong - 1) / kLong, ends = to / kLong;
    const bool any_whole = !FEW && whole < ends;
    const int head = any_whole ? whole * kLong - from : to - from, stretches = any_whole ? ends - whole : 0, tail = any_whole ? to - ends * kLong : 0;
    for (int v0 = 0; v0 < vectors; v0 += a.lanes) {
      const int d = vector_at<VE>(min(v0 + lane, vectors - 1), a.num_dims);
      float sum[VE] = {};
      if (stretches > 0)
        sum_items_together<float, VE>(stretches, a.lanes, [&](int i) {
          return reinterpret_cast<const LoosePack<float, VE>*>(a.long_sums + (long long)(whole + i) * a.num_dims + d);
        }, sum, parts);
      sum_items_together<T, VE>(head + tail, a.lanes, [&](int i) {
        const int at = i < head ? from + i : ends * kLong + i - head;
        return reinterpret_cast<const LoosePack<T, VE>*>(grad + (long long)(FEW ? in_order[at] : a.places[at]) * a.grad_stride + d);
      }, sum, parts);
      if (tid < a.lanes) store<STREAMED>(out + (long long)r * a.num_dims + d, sum, a.scale);
    }
  }
}

struct GradScratch {
  int *keys[2], *places[2], *counts;
  float* long_sums;
  int* bounds;
  size_t bytes;
  GradScratch(void* memory, long long num_ids, long long num_rows, int num_dims, const SortPlan& p) {
    WorkspaceParts s(memory);
    for (int i = 0; i < 2; ++i) {
      keys[i] = s.part<int>((size_t)num_ids);
      places[i] = s.part<int>((size_t)num_ids);
    }
    counts = s.part<int>((size_t)p.blocks << p.bits);
    long_sums = s.part<float>((size_t)(num_ids / kLong) * num_dims);
    bounds = s.part<int>((size_t)num_rows / 4 + 2);  // (every workgroup but the last has four rows or more: one for each group of lanes)
    bytes = s.used();
  }
};

}  // namespace cuhnsw_amd

using namespace cuhnsw_amd;

extern "C" {

int cuhnsw_use_device(int device, int* before) {
  int now = -1;
  if (!before || hipGetDevice(&now) != hipSuccess || (now != device && hipSetDevice(device) != hipSuccess)) {
    (void)hipGetLastError();
    set_call_error("no such HIP device");
    return -1;
  }
  *before = now;
  return 0;
}

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
  if (num_ids <= kFew || num_ids > 1 << 30 || num_rows <= 0 || num_rows >= 0x7fffffff || num_dims <= 0) return 0;
  return (long long)GradScratch(nullptr, num_ids, num_rows, num_dims, sort_plan(num_ids, num_rows)).bytes;
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
    GradArgs g{};
    g.grad = grad;
    g.grad_stride = grad_stride;
    g.ids = ids;
    g.ids_64 = ids_64;
    g.num_ids = (int)num_ids;
    g.num_rows = (int)num_rows;
    g.num_dims = num_dims;
    g.scale = scale;
    g.out = out;
    const bool few = num_ids <= kFew;
    const SortPlan p = sort_plan(num_ids, num_rows);
    const GradScratch w(few ? nullptr : workspace, num_ids, num_rows, num_dims, p);
    if (!few) {
      want(workspace && workspace_bytes >= (long long)w.bytes, "lookup gradient: the workspace is too small");
      g.keys = w.keys[(p.passes - 1) & 1];
      g.places = w.places[(p.passes - 1) & 1];
      g.long_sums = w.long_sums;
      g.bounds = w.bounds;
      g.num_stretches = (int)(num_ids / kLong);
    }
    auto sort_ids = [&] {
      for (int pass = 0; pass < p.passes; ++pass) {
        const SortInput in{ids, ids_64, (int)num_rows, pass ? w.keys[(pass - 1) & 1] : nullptr, pass ? w.places[(pass - 1) & 1] : nullptr};
        hipLaunchKernelGGL(sort_count_kernel, dim3(p.blocks), dim3(kSortThreads), 0, s, in, (int)num_ids, p.chunk, pass * p.bits, 1 << p.bits,
                           w.counts);
        hipLaunchKernelGGL(sort_place_kernel, dim3(p.blocks), dim3(kSortThreads), 0, s, in, (int)num_ids, p.chunk, pass * p.bits, 1 << p.bits,
                           p.bits, w.counts, w.keys[pass & 1], w.places[pass & 1]);
      }
      HIP_CHECK(hipGetLastError());
    };
    with_type(grad_type, [&](auto* t) {
      with_type(out_type, [&](auto* u) {
        using T = std::remove_pointer_t<decltype(t)>;
        using U = std::remove_pointer_t<decltype(u)>;
        if constexpr (std::is_same_v<T, U> || std::is_same_v<T, float>) {
          with_vector<T>(num_dims, [&](auto ve) {
            constexpr int VE = decltype(ve)::value;
            g.lanes = lanes_of(vectors_of<VE>(num_dims));
            // rows for about 32 KB in and out, whole turns of the groups of lanes
            const int groups = 256 / g.lanes;
            const long long bytes = (long long)num_dims * (sizeof(U) + sizeof(T) * (num_ids / num_rows));
            g.rows = (int)std::min<long long>(kMostRows, std::max<long long>(groups, 32768 / bytes / groups * groups));
            g.num_blocks = (int)((num_rows + g.rows - 1) / g.rows);
            if (!few) {
              sort_ids();
              in_launches(g, (long long)g.num_stretches + g.num_blocks / 256 + 1,
                          [&](dim3 grid) { hipLaunchKernelGGL((grad_long_kernel<T, VE>), grid, dim3(256), 0, s, g); });
            }
            with_flag(num_rows * num_dims * (long long)sizeof(U) >= kStreamedFrom, [&](auto streamed) {
              constexpr bool kStreamed = decltype(streamed)::value;
              in_launches(g, g.num_blocks, [&](dim3 grid) {
                if (few) hipLaunchKernelGGL((grad_kernel<T, U, VE, true, kStreamed>), grid, dim3(256), (size_t)num_ids * 12, s, g);
                else hipLaunchKernelGGL((grad_kernel<T, U, VE, false, kStreamed>), grid, dim3(256), 0, s, g);
              });
            });
          });
        } else {
          throw std::runtime_error("lookup gradient: the gradient has the table's type or is float32");
        }
      });
    });
  });
}

}  // extern "C"
