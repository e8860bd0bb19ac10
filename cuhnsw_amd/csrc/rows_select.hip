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

constexpr int kMostNum = 256, kMostBeams = 1024, kMostLists = 4096;
constexpr int kThreads = 256, kWaves = 4;
constexpr int kKept = 2048;  // candidates a workgroup holds in LDS

struct SelectArgs {
  const void* scores;
  long long stride_b, stride_k;
  int num_batch, num_beams, num_values;
  const float* beams;             // [num_batch, num_beams] or null
  const unsigned char* finished;  // the same, or null
  int normalise, end, num;
  float* out_totals;
  int *out_parents, *out_tokens;
  int parts, each;     // workgroups of a row, tiles of each of them
  int most;            // min(num, num_values)
  uint64_t* lists;     // per row and part: its `most` best, largest first; 0 where there are not so many
  float* list_top;     // per row and part: the largest score,
  double* list_sum;    // and the sum of exp(score - largest)
};

// Orders as the values do, +0 and -0 as one; larger keys first means lower places first among equals.  No key is 0.
__device__ inline uint64_t order_key(float x, uint32_t place) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~place;
}
__device__ inline float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ inline int key_place(uint64_t key) { return (int)~(uint32_t)key; }
__device__ inline float score_at(float x) { return fmaxf(x, -INFINITY); }  // (of a NaN: the other operand)

// The num-th largest of the workgroup's threads' values, by counting: of the values that fewer than num are above, the
// smallest.  `all` has a place for every thread.
template <typename T>
__device__ inline T reached_by(T mine, int num, T largest_possible, T* all) {
  all[threadIdx.x] = mine;
  __syncthreads();
  int above = 0;
#pragma unroll 8
  for (int i = 0; i < kThreads; ++i) above += all[i] > mine;
  T least = above < num ? mine : largest_possible;
  for (int step = 32; step > 0; step >>= 1) {
    const T other = __shfl_xor(least, step);
    least = other < least ? other : least;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) all[threadIdx.x >> 6] = least;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) least = all[w] < least ? all[w] : least;
  return least;
}

// The best of `count` different keys to the front, in order; how many there are then (at most `most`).  Up to two for every thread are
// ranked by counting the larger ones, more go through a bitonic network.
__device__ inline int keep_best(uint64_t* keys, int count, int most) {
  const int tid = threadIdx.x;
  __syncthreads();
  if (count <= 2 * kThreads) {
    uint64_t mine[2];
    int rank[2] = {0, 0};
    for (int j = 0; j < 2; ++j) mine[j] = tid + j * kThreads < count ? keys[tid + j * kThreads] : 0;
    if (count <= kThreads) {
#pragma unroll 8
      for (int i = 0; i < count; ++i) rank[0] += keys[i] > mine[0];
    } else {
#pragma unroll 8
      for (int i = 0; i < count; ++i) {
        const uint64_t other = keys[i];
        rank[0] += other > mine[0];
        rank[1] += other > mine[1];
      }
    }
    __syncthreads();
    for (int j = 0; j < 2; ++j)
      if (mine[j] && rank[j] < most) keys[rank[j]] = mine[j];
  } else {
    int size = 1024;
    while (size < count) size <<= 1;
    for (int i = count + tid; i < size; i += kThreads) keys[i] = 0;
    for (int run = 2; run <= size; run <<= 1)
      for (int step = run >> 1; step > 0; step >>= 1) {
        __syncthreads();
        for (int i = tid; i < size / 2; i += kThreads) {
          const int a = (i / step) * 2 * step + i % step, b = a + step;
          const uint64_t x = keys[a], y = keys[b];
          if ((x < y) == ((a & run) == 0)) {
            keys[a] = y;
            keys[b] = x;
          }
        }
      }
  }
  __syncthreads();
  return min(count, most);
}

// Pass over a row's scores: NV vectors of 16 bytes for each thread are a tile, and the next tile is asked for before the one
// at hand is looked at.  The first tile gives a value that `num` of its scores reach; a score that is not below it goes to a list in
// LDS.  After 1, 2, 4, 8... tiles the list is cut down to its best, and what comes later has to reach the worst of them: a hundred
// or so enter between two cuts, and between two cuts the wavefronts do not wait for each other.  Where a list would
// overflow meanwhile (scores in an order that is hard) those tiles are gone over again, a score of each thread at a time.
//
// What a score costs: its conversion, a comparison, and normalised the maximum, a subtraction, a product, the exponential (of four
// times the cost) and an addition.
template <typename T, int NV, bool NORMALISE>
__global__ void __launch_bounds__(kThreads, 6) select_part_kernel(SelectArgs a) {
  constexpr int VE = 16 / sizeof(T), EACH = NV * VE;
  typedef LoosePack<T, VE> Vector;
  __shared__ uint64_t kept[kKept];
  __shared__ float shared[kThreads];
  __shared__ double shared_sum[kWaves];
  __shared__ int filled;
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts, b = row / a.num_beams, k = row - b * a.num_beams;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (a.finished && a.finished[row]) return;
  const T* x = static_cast<const T*>(a.scores) + b * a.stride_b + k * a.stride_k;
  // Whole vectors of the row, wherever it begins (global memory takes 16 bytes from any address), and the scores behind them,
  // which the first workgroup of the row takes one by one.  Which thread gets which score depends on the sizes alone: equal
  // rows have the same sum to the last bit, and equal candidates of theirs are equal.
  const int vectors = a.num_values / VE, tail = a.num_values - vectors * VE;
  if (tid == 0) filled = 0;
  __syncthreads();
  constexpr int kTile = kThreads * NV;  // vectors
  auto load = [&](int first, Vector (&to)[NV]) {
    const T* from = x + (first + tid) * VE;
    if (first + kTile <= vectors) {
#pragma unroll
      for (int i = 0; i < NV; ++i) to[i] = *reinterpret_cast<const Vector*>(from + i * (kThreads * VE));
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < VE; ++j) to[i].at[j] = narrow<T>(-INFINITY);
        if (first + i * kThreads + tid < vectors) to[i] = *reinterpret_cast<const Vector*>(from + i * (kThreads * VE));
      }
    }
  };
  int have = 0;
  uint64_t bar_key = 0;  // what a key has to be above, once the list was cut
  float bar = 0.f;       // what a score has to reach (always finite: -infinity and NaN never do)
  constexpr float kLowest = -3.402823466e38f;
  auto cut = [&] {
    have = keep_best(kept, have, a.most);
    if (have == a.most) {
      bar_key = kept[have - 1];
      bar = fmaxf(key_value(bar_key), kLowest);
    }
    if (tid == 0) filled = have;
    __syncthreads();
  };
  float top = -INFINITY, sum = 0.f;
  const int first_vector = part * a.each * kTile;
  const int tiles = max(part == 0 ? 1 : 0, first_vector < vectors ? min(a.each, (vectors - first_vector + kTile - 1) / kTile) : 0);
  const int extra_place = vectors * VE + tid;
  const float extra = part == 0 && tid < tail ? score_at(widen(x[extra_place])) : -INFINITY;
  auto place = [&](int t, int i) { return (first_vector + t * kTile + i / VE * kThreads + tid) * VE + i % VE; };
  Vector next[NV];
  if (tiles > 0) load(first_vector, next);
  for (int t = 0, segment = 1; t < tiles; segment = t) {
    const int begin = t, end = min(tiles, t + segment);
    for (; t < end; ++t) {
      float v[EACH];
#pragma unroll
      for (int i = 0; i < EACH; ++i) v[i] = NORMALISE ? score_at(widen(next[i / VE].at[i % VE])) : widen(next[i / VE].at[i % VE]);
      if (t + 1 < tiles) load(first_vector + (t + 1) * kTile, next);
      if (NORMALISE || t == 0) {
        float largest = t == 0 ? extra : -INFINITY;
#pragma unroll
        for (int i = 0; i < EACH; ++i) largest = fmaxf(largest, v[i]);
        if (NORMALISE) {
          constexpr float kLog2e = 1.44269504f;
          if (largest > top) {
            sum *= __builtin_amdgcn_exp2f((top - largest) * kLog2e);
            top = largest;
          }
          const float base = top == -INFINITY ? 0.f : top, before = sum;
          if (t == 0) sum += __builtin_amdgcn_exp2f((extra - base) * kLog2e);
#pragma unroll
          for (int i = 0; i < EACH; ++i) sum += __builtin_amdgcn_exp2f((v[i] - base) * kLog2e);
          if (top == INFINITY) {  // (beside an infinite one only the infinite ones count)
            sum = before + (t == 0 && extra == INFINITY ? 1.f : 0.f);
            for (int i = 0; i < EACH; ++i) sum += v[i] == INFINITY ? 1.f : 0.f;
          }
        }
        if (t == 0) bar = fmaxf(reached_by(largest, a.most, INFINITY, shared), kLowest);
      }
      auto offer = [&](float value, int at_row) {
        const bool in = value >= bar;
        const unsigned long long with = __ballot(in);
        if (with) {
          int at = 0;
          if (lane == 0) at = atomicAdd(&filled, __popcll(with));
          at = __shfl(at, 0) + __popcll(with & ((1ull << lane) - 1));
          if (in && at < kKept) kept[at] = order_key(value, (uint32_t)at_row);
        }
      };
#pragma unroll
      for (int i = 0; i < EACH; ++i) offer(v[i], place(t, i));
      if (t == 0) offer(extra, extra_place);
    }
    __syncthreads();
    if (filled <= kKept) {
      have = filled;
    } else {
      for (int again = begin; again < end; ++again)
        for (int i = 0; i < EACH + (again == 0 ? 1 : 0); ++i) {
          if ((again == begin && i == 0) || have + kThreads > kKept) cut();
          const int at_row = i < EACH ? place(again, i) : extra_place;
          const bool there = i < EACH ? first_vector + again * kTile + i / VE * kThreads + tid < vectors : part == 0 && tid < tail;
          const float value = there ? score_at(widen(x[at_row])) : -INFINITY;
          const uint64_t key = order_key(value, (uint32_t)at_row);
          if (value > -INFINITY && key > bar_key) kept[atomicAdd(&filled, 1)] = key;
          __syncthreads();
          have = filled;
          __syncthreads();
        }
    }
    if (t < tiles && have > a.most) cut();
    __syncthreads();
  }
  have = keep_best(kept, have, a.most);
  uint64_t* list = a.lists + (long long)blockIdx.x * a.most;
  for (int i = tid; i < a.most; i += kThreads) list[i] = i < have ? kept[i] : 0;
  if (NORMALISE) {
    float most = top;
    for (int step = 32; step > 0; step >>= 1) most = fmaxf(most, __shfl_xor(most, step));
    if (lane == 0) shared[wave] = most;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) most = fmaxf(most, shared[w]);
    double part_sum = top == most ? (double)sum : sum * exp((double)top - (double)most);
    if (top == -INFINITY) part_sum = 0.0;
    for (int step = 32; step > 0; step >>= 1) part_sum += __shfl_xor(part_sum, step);
    if (lane == 0) shared_sum[wave] = part_sum;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWaves; ++w) part_sum += shared_sum[w];
      a.list_top[blockIdx.x] = most;
      a.list_sum[blockIdx.x] = part_sum;
    }
  }
}

// Orders as the values do; 0 is below all of them.
__device__ inline uint64_t order_total(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u & 0x8000000000000000ull ? ~u : u | 0x8000000000000000ull;
}
__device__ inline double total_value(uint64_t u) {
  return __longlong_as_double((long long)(u & 0x8000000000000000ull ? u & 0x7fffffffffffffffull : ~u));
}

// The lists of a batch entry's beams and parts become its answer: the totals in 64 bits, those that num of the threads' best
// reach in LDS, each ranked among them by (total, lower beam, its own order).
__global__ void __launch_bounds__(kThreads) select_merge_kernel(SelectArgs a) {
  __shared__ uint64_t kept_total[kKept], kept_key[kKept];
  __shared__ int kept_beam[kKept];
  __shared__ uint64_t shared[kThreads];
  __shared__ int filled, first_best;
  extern __shared__ double beam_less[];  // per beam: the logarithm of its sum, and its largest score behind
  double* beam_top = beam_less + a.num_beams;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int per_beam = a.parts * a.most, all = a.num_beams * per_beam;
  for (int k = tid >> 6; a.normalise && k < a.num_beams; k += kWaves) {
    const long long row = (long long)b * a.num_beams + k;
    if (a.finished && a.finished[row]) continue;
    float top = -INFINITY;
    for (int p = lane; p < a.parts; p += 64) top = fmaxf(top, a.list_top[row * a.parts + p]);
    for (int step = 32; step > 0; step >>= 1) top = fmaxf(top, __shfl_xor(top, step));
    double sum = 0.0;
    for (int p = lane; p < a.parts; p += 64) {
      const float t = a.list_top[row * a.parts + p];
      const double s = a.list_sum[row * a.parts + p];
      if (t > -INFINITY) sum += t == top ? s : s * exp((double)t - (double)top);
    }
    for (int step = 32; step > 0; step >>= 1) sum += __shfl_xor(sum, step);
    if (lane == 0) {
      beam_top[k] = top;
      beam_less[k] = log(sum);
    }
  }
  if (tid == 0) filled = 0;
  __syncthreads();
  auto key_of = [&](int c) { return a.lists[(long long)b * all + c]; };
  auto total_of = [&](int c, uint64_t key) -> uint64_t {  // 0: no candidate
    const int k = c / per_beam;
    const long long row = (long long)b * a.num_beams + k;
    const double beam = a.beams ? a.beams[row] : 0.f;
    double total;
    if (a.finished && a.finished[row]) {
      if (c != k * per_beam) return 0;
      total = beam;
    } else {
      if (key == 0) return 0;
      total = key_value(key);
      if (a.normalise) total = (total == beam_top[k] ? 0.0 : total - beam_top[k]) - beam_less[k];
      total += beam;
    }
    return total > -INFINITY ? order_total(total) : 0;
  };
  constexpr int kHeld = 4;  // candidates of a thread that stay in registers
  uint64_t best = 0, keys[kHeld], totals[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) keys[i] = tid + i * kThreads < all ? key_of(tid + i * kThreads) : 0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    totals[i] = tid + i * kThreads < all ? total_of(tid + i * kThreads, keys[i]) : 0;
    best = totals[i] > best ? totals[i] : best;
  }
  for (int c = tid + kHeld * kThreads; c < all; c += kThreads) {
    const uint64_t t = total_of(c, key_of(c));
    best = t > best ? t : best;
  }
  const uint64_t bar = reached_by(best, a.num, ~(uint64_t)0, shared);
  auto offer = [&](int c, uint64_t key, uint64_t t) {
    if (t == 0 || t < bar) return;
    const int at = atomicAdd(&filled, 1);
    if (at >= kKept) return;
    const int k = c / per_beam;
    kept_total[at] = t;
    kept_key[at] = a.finished && a.finished[(long long)b * a.num_beams + k] ? (uint64_t)(uint32_t)~(uint32_t)a.end : key;
    kept_beam[at] = k;
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) offer(tid + i * kThreads, keys[i], totals[i]);
  if (best >= bar)
    for (int c = tid + kHeld * kThreads; c < all; c += kThreads) {
      const uint64_t key = key_of(c);
      offer(c, key, total_of(c, key));
    }
  __syncthreads();
  const int count = filled;
  const long long out = (long long)b * a.num;
  if (count <= kKept) {
    for (int i = tid; i < count; i += kThreads) {
      const uint64_t t = kept_total[i], key = kept_key[i];
      const int k = kept_beam[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < count; ++j) {
        const uint64_t other = kept_total[j];
        if (other == t) rank += kept_beam[j] < k || (kept_beam[j] == k && kept_key[j] > key);
        else rank += other > t;
      }
      if (rank < a.num) {
        a.out_totals[out + rank] = (float)total_value(t);
        a.out_parents[out + rank] = k;
        a.out_tokens[out + rank] = key_place(key);
      }
    }
    for (int i = count + tid; i < a.num; i += kThreads) {
      a.out_totals[out + i] = -INFINITY;
      a.out_parents[out + i] = a.out_tokens[out + i] = -1;
    }
    return;
  }
  // More equal totals than are held: one after the other, each the best of those behind the last one.
  uint64_t last = ~0ull, last_key = 0;
  int last_beam = -1;
  for (int i = 0; i < a.num; ++i) {
    uint64_t mine = 0, mine_key = 0;
    int mine_beam = 0;
    auto before = [](uint64_t t, int k, uint64_t key, uint64_t t2, int k2, uint64_t key2) {
      return t != t2 ? t > t2 : k != k2 ? k < k2 : key > key2;
    };
    for (int c = tid; c < all; c += kThreads) {
      const int k = c / per_beam;
      uint64_t key = key_of(c);
      const uint64_t t = total_of(c, key);
      if (t == 0) continue;
      if (a.finished && a.finished[(long long)b * a.num_beams + k]) key = (uint64_t)(uint32_t)~(uint32_t)a.end;
      if (last_beam >= 0 && !before(last, last_beam, last_key, t, k, key)) continue;
      if (mine == 0 || before(t, k, key, mine, mine_beam, mine_key)) mine = t, mine_key = key, mine_beam = k;
    }
    for (int step = 1; step < 64; step <<= 1) {
      const uint64_t t = __shfl_xor(mine, step), key = __shfl_xor(mine_key, step);
      const int k = __shfl_xor(mine_beam, step);
      if (t != 0 && (mine == 0 || before(t, k, key, mine, mine_beam, mine_key))) mine = t, mine_key = key, mine_beam = k;
    }
    __syncthreads();
    if (lane == 0) kept_total[tid >> 6] = mine, kept_key[tid >> 6] = mine_key, kept_beam[tid >> 6] = mine_beam;
    __syncthreads();
    if (tid == 0) {
      int w = 0;
      for (int o = 1; o < kWaves; ++o)
        if (kept_total[o] != 0 && (kept_total[w] == 0 || before(kept_total[o], kept_beam[o], kept_key[o], kept_total[w], kept_beam[w], kept_key[w]))) w = o;
      first_best = w;
      const bool there = kept_total[w] != 0;
      a.out_totals[out + i] = there ? (float)total_value(kept_total[w]) : -INFINITY;
      a.out_parents[out + i] = there ? kept_beam[w] : -1;
      a.out_tokens[out + i] = there ? key_place(kept_key[w]) : -1;
    }
    __syncthreads();
    last = kept_total[first_best];
    last_key = kept_key[first_best];
    last_beam = kept_beam[first_best];
    if (last == 0) {  // (nothing is left)
      for (int j = i + 1 + tid; j < a.num; j += kThreads) {
        a.out_totals[out + j] = -INFINITY;
        a.out_parents[out + j] = a.out_tokens[out + j] = -1;
      }
      return;
    }
  }
}

// ----------------------------------------------------------------------------------------------- states
constexpr int kMostStates = 32;
struct ReorderArgs {
  const unsigned char* from[kMostStates];
  unsigned char* to[kMostStates];
  long long stride_b[kMostStates], stride_k[kMostStates], bytes[kMostStates];  // in bytes; the results are dense
  unsigned char width[kMostStates];  // bytes that move together: the widest that sizes, strides and addresses allow
  const int* parents;
  long long parent_stride_b, parent_stride_k;
  int num_beams, num_picked;
};

template <typename T>
__device__ inline void copy_or_clear(const unsigned char* from, unsigned char* to, long long bytes, bool there) {
  const long long n = bytes / (long long)sizeof(T), stride = (long long)gridDim.x * 256;
  const T* in = reinterpret_cast<const T*>(from);
  T* out = reinterpret_cast<T*>(to);
  long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (!there) {
    for (; i < n; i += stride) out[i] = T{};
    return;
  }
  for (; i + 3 * stride < n; i += 4 * stride) {
    const T a = in[i], b = in[i + stride], c = in[i + 2 * stride], d = in[i + 3 * stride];
    out[i] = a;
    out[i + stride] = b;
    out[i + 2 * stride] = c;
    out[i + 3 * stride] = d;
  }
  for (; i < n; i += stride) out[i] = in[i];
}

__global__ void __launch_bounds__(256) reorder_kernel(ReorderArgs a) {
  const int s = blockIdx.z, row = blockIdx.y, b = row / a.num_picked, j = row - b * a.num_picked;
  const int parent = a.parents[b * a.parent_stride_b + j * a.parent_stride_k];
  const bool there = parent >= 0 && parent < a.num_beams;
  const unsigned char* from = a.from[s] + b * a.stride_b[s] + (there ? parent : 0) * a.stride_k[s];
  unsigned char* to = a.to[s] + row * a.bytes[s];
  switch (a.width[s]) {
    case 16: copy_or_clear<uint4>(from, to, a.bytes[s], there); break;
    case 8: copy_or_clear<uint2>(from, to, a.bytes[s], there); break;
    case 4: copy_or_clear<uint32_t>(from, to, a.bytes[s], there); break;
    case 2: copy_or_clear<uint16_t>(from, to, a.bytes[s], there); break;
    default: copy_or_clear<uint8_t>(from, to, a.bytes[s], there); break;
  }
}

// How a selection is spread: tiles of one vector or of 16 scores for each thread, and so many workgroups a row as the machine
// holds at once (six on a CU: one more would be a second round).
constexpr int kResident = 6 * 256;
struct SelectPlan {
  bool small;
  int parts, each;
};
static SelectPlan select_plan(int type, int num_batch, int num_beams, int num_values, int num) {
  SelectPlan p;
  const long long rows = (long long)num_batch * num_beams;
  const int most = std::min(num, num_values);
  p.small = rows * num_values < 512ll * 8192;
  const long long tile = kThreads * (p.small ? 16 / (long long)element_size(type) : 16);
  const int tiles = (int)((num_values + tile - 1) / tile);
  const long long wanted = std::min<long long>({std::max<long long>(1, kResident / rows), 256, std::max<long long>(1, 16384 / ((long long)num_beams * most))});
  p.each = (int)((tiles + wanted - 1) / wanted);
  p.parts = (tiles + p.each - 1) / p.each;
  return p;
}

struct SelectScratch {
  uint64_t* lists;
  double* sums;
  float* tops;
  size_t bytes;
  SelectScratch(void* memory, long long rows, int parts, int most) {
    WorkspaceParts s(memory);
    lists = s.part<uint64_t>((size_t)rows * parts * most);
    sums = s.part<double>((size_t)rows * parts);
    tops = s.part<float>((size_t)rows * parts);
    bytes = s.used();
  }
};

}  // namespace cuhnsw_amd

using namespace cuhnsw_amd;

extern "C" {

long long cuhnsw_select_beams_workspace(int type, int num_batch, int num_beams, int num_values, int num) {
  if (!known_type(type) || num_batch <= 0 || num_beams <= 0 || num_values <= 0 || num <= 0) return 0;
  return (long long)SelectScratch(nullptr, (long long)num_batch * num_beams, select_plan(type, num_batch, num_beams, num_values, num).parts,
                                  std::min(num, num_values)).bytes;
}

int cuhnsw_select_beams(const void* scores, int type, long long stride_b, long long stride_k, int num_batch, int num_beams, int num_values,
                        const float* beams, const unsigned char* finished, int end, int normalise, int num, float* out_totals,
                        int* out_parents, int* out_tokens, void* workspace, long long workspace_bytes, void* stream) {
  return call_guarded([&] {
    want(known_type(type), "select: unknown element type");
    want(num_batch >= 0 && num_beams > 0 && num_values > 0, "select: bad sizes");
    want(num_values <= 1 << 30, "select: more than 2^30 values");
    want(num > 0 && num <= kMostNum, "select: between 1 and 256 candidates can be asked for");
    want((long long)num_beams * std::min(num, num_values) <= kMostLists, "select: more than 4096 candidates of all beams (beams times candidates asked for)");
    want(num_beams <= kMostBeams, "select: more than 1024 beams");
    want((long long)num_batch * num_beams <= 0x7fffffff, "select: too many rows");
    if (num_batch == 0) return;
    want(scores && out_totals && out_parents && out_tokens, "select: null argument");
    want(!finished || (end >= 0 && end < num_values), "select: the token that ends a sequence is outside the vocabulary");
    const SelectPlan p = select_plan(type, num_batch, num_beams, num_values, num);
    const long long rows = (long long)num_batch * num_beams;
    const SelectScratch w(workspace, rows, p.parts, std::min(num, num_values));
    want(workspace && workspace_bytes >= (long long)w.bytes, "select: the workspace is too small");
    want(rows * p.parts <= 0x7fffffff, "select: too many rows");
    const SelectArgs a{scores, stride_b, stride_k, num_batch, num_beams, num_values, beams, finished, normalise, end, num,
                       out_totals, out_parents, out_tokens, p.parts, p.each, std::min(num, num_values), w.lists, w.tops, w.sums};
    hipStream_t s = static_cast<hipStream_t>(stream);
    with_type(type, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      const dim3 grid((unsigned)(rows * p.parts));
      if (p.small && normalise) hipLaunchKernelGGL((select_part_kernel<T, 1, true>), grid, dim3(kThreads), 0, s, a);
      else if (p.small) hipLaunchKernelGGL((select_part_kernel<T, 1, false>), grid, dim3(kThreads), 0, s, a);
      else if (normalise) hipLaunchKernelGGL((select_part_kernel<T, sizeof(T), true>), grid, dim3(kThreads), 0, s, a);
      else hipLaunchKernelGGL((select_part_kernel<T, sizeof(T), false>), grid, dim3(kThreads), 0, s, a);
    });
    hipLaunchKernelGGL(select_merge_kernel, dim3((unsigned)num_batch), dim3(kThreads), (size_t)num_beams * 16, s, a);
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
        const uint64_t all = (uint64_t)a.bytes[i] | (uint64_t)a.stride_b[i] | (uint64_t)a.stride_k[i] | reinterpret_cast<uintptr_t>(a.from[i]) |
                             reinterpret_cast<uintptr_t>(a.to[i]) | 16;
        a.width[i] = (unsigned char)(all & (~all + 1));
        most = std::max(most, a.bytes[i] / a.width[i]);
      }
      if (most == 0) continue;
      a.parents = parents;
      a.parent_stride_b = parent_stride_b;
      a.parent_stride_k = parent_stride_k;
      a.num_beams = num_beams;
      a.num_picked = num_picked;
      hipLaunchKernelGGL(reorder_kernel, dim3((unsigned)std::min<long long>((most + 1023) / 1024, 256), (unsigned)(num_batch * num_picked), (unsigned)count),
                         dim3(256), 0, static_cast<hipStream_t>(stream), a);
      HIP_CHECK(hipGetLastError());
    }
  });
}

}  // extern "C"
