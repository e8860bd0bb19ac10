// The best candidates over the beams of a search and a vocabulary, and the reordering of the beams' states that follows.
//
//   total[b][k][v] = beams[b][k] + x[b][k][v]                                     as the scores are
//   total[b][k][v] = beams[b][k] + x[b][k][v] - log(sum over u of exp(x[b][k][u]))  normalised
//   the `num` largest totals of b over (k, v), largest first; of equal ones the lower k first, then the larger x, then the
//   lower v.
//
// Totals are formed, held and compared in 64 bits; the sum in them is one of the machine's exponentials in float32, joined in 64
// bits, and good to about 2^-20 of itself: candidates of different beams whose totals are nearer than that may stand in either
// order, those of one beam stand in the scores' own.  A NaN counts as -infinity, and what is -infinity is never chosen: places that are
// left over say -infinity, parent -1, token -1.  Where a score is +infinity the formula has no value, and only the beam's n
// infinite ones are candidates, each with total beams[b][k] - log(n).  A finished beam has one candidate, the token `end` with
// the beam's own score.
#include <algorithm>

#include "../../include/cuhnsw_amd.h"
#include "rows.h"

namespace cuhnsw_amd {

constexpr int kMostNum = 256, kMostBeams = 1024, kMostLists = 4096;
constexpr int kMostCandidates = 16384;  // in the lists of a batch entry: what one workgroup holds in registers
constexpr int kThreads = 256, kWaves = 4, kEach = 16;
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
__device__ inline float reached_by(float mine, int num, float* all) {
  all[threadIdx.x] = mine;
  __syncthreads();
  int above = 0;
#pragma unroll 8
  for (int i = 0; i < kThreads; ++i) above += all[i] > mine;
  float least = above < num ? mine : INFINITY;
  for (int step = 32; step > 0; step >>= 1) {
    least = fminf(least, __shfl_xor(least, step));
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) all[threadIdx.x >> 6] = least;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) least = fminf(least, all[w]);
  return least;
}

// The best of `count` different keys to the front, in order; how many there are then (at most `most`).  Up to two for every thread are
// ranked by counting the larger ones.  Of more (up to kKept) those are picked first that reach a bar which enough of them
// reach and no more than that: it is found by halving, with the keys in registers.
__device__ inline int keep_best(uint64_t* keys, int count, int most, int (&counts)[2][kWaves]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __syncthreads();
  if (count > 2 * kThreads) {
    constexpr int kMine = kKept / kThreads;
    uint64_t mine[kMine], bar = 1, beyond = ~0ull;
#pragma unroll
    for (int i = 0; i < kMine; ++i) mine[i] = tid + i * kThreads < count ? keys[tid + i * kThreads] : 0;
    int turn = 0, before;
    for (uint64_t probe = beyond / 2;; probe = bar + (beyond - bar) / 2, turn ^= 1) {
      int reach = 0;
#pragma unroll
      for (int i = 0; i < kMine; ++i) reach += __popcll(__ballot(mine[i] >= probe));
      if (lane == 0) counts[turn][wave] = reach;
      __syncthreads();
      reach = before = 0;
      for (int w = 0; w < kWaves; ++w) {
        before += w < wave ? counts[turn][w] : 0;
        reach += counts[turn][w];
      }
      if (reach < most) {
        beyond = probe;
      } else {
        bar = probe;
        count = reach;
        if (count <= 2 * kThreads) break;
      }
    }
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const unsigned long long with = __ballot(mine[i] >= bar);
      if (mine[i] >= bar) keys[before + __popcll(with & ((1ull << lane) - 1))] = mine[i];
      before += __popcll(with);
    }
    __syncthreads();
  }
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
  __syncthreads();
  return min(count, most);
}

// Pass over a row's scores: 16 for each thread are a tile, in vectors of 16 bytes, and the next tile is asked for before the
// one at hand is looked at.  The first tile gives a value that `num` of its scores reach; a score that is not below it goes to a list in
// LDS.  After 1, 2, 4, 8... tiles the list is cut down to its best, and what comes later has to reach the worst of them: a hundred
// or so enter between two cuts, and between two cuts the wavefronts do not wait for each other.  Where a list would
// overflow meanwhile (scores in an order that is hard) those tiles are gone over again, a score of each thread at a time.
//
// What a score costs: its conversion, a comparison, and normalised the maximum, a subtraction, a product, the exponential (of four
// times the cost) and an addition.  100 rows of 1 183 514 float32, the best 100: 103 us, 4.6 TB/s of reads;
// 32 x 8 rows of 131 072 bfloat16, normalised: 34 us, 2.0 TB/s, bound by these instructions.
//
// (Tiles of 4 float32 for each thread instead of 16 are up to 0.5 us faster where rows are few and short, 5 of 28 slower at 128
// rows of 32 000, 6 of 45 at one of 1 000 000.)
template <typename T, bool NORMALISE>
__global__ void __launch_bounds__(kThreads, 6) select_part_kernel(SelectArgs a) {
  constexpr int VE = 16 / sizeof(T), EACH = kEach, NV = EACH / VE;
  typedef LoosePack<T, VE> Vector;
  __shared__ uint64_t kept[kKept];
  __shared__ float shared[kThreads];
  __shared__ double shared_sum[kWaves];
  __shared__ int filled, counts[2][kWaves];
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
    have = keep_best(kept, have, a.most, counts);
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
          const float base = top == -INFINITY ? 0.f : top;
          float of_tile = t == 0 ? __builtin_amdgcn_exp2f((extra - base) * kLog2e) : 0.f;
#pragma unroll
          for (int i = 0; i < EACH; ++i) of_tile += __builtin_amdgcn_exp2f((v[i] - base) * kLog2e);
          if (top == INFINITY) {  // (beside an infinite one only the infinite ones count)
            of_tile = t == 0 && extra == INFINITY ? 1.f : 0.f;
            for (int i = 0; i < EACH; ++i) of_tile += v[i] == INFINITY ? 1.f : 0.f;
          }
          sum += of_tile;
        }
        if (t == 0) bar = fmaxf(reached_by(largest, a.most, shared), kLowest);
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
  have = keep_best(kept, have, a.most, counts);
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

// The lists of a batch entry's beams and parts become its answer: the totals in 64 bits, all of them in registers; a bar that at
// least num of them reach and not many more; those in LDS, each ranked there by (total, lower beam, its own order).  Four lanes
// count for one value.  One workgroup for each batch entry, and what it does is a chain of short steps, each of which waits for the
// one before: 10 us for a handful of candidates, 14 with the sums of 8 beams, 22 and 34 for 12 000 and 16 000 candidates.
constexpr int kMerge = 1024, kMergeWaves = kMerge / 64, kGroups = kMerge / 4;

// HELD: candidates of a thread.  Few ones' code is a third of the other's, and it is read from memory at every call: what it saved
// is beside the plan.
template <int HELD>
__global__ void __launch_bounds__(kMerge) select_merge_kernel(SelectArgs a) {
  __shared__ uint64_t kept_total[kKept], kept_key[kKept];
  __shared__ int kept_beam[kKept];
  __shared__ uint64_t group_best[kGroups];
  __shared__ int counts[2][kMergeWaves];
  __shared__ int filled, first_best;
  extern __shared__ double beam_less[];  // per beam: the logarithm of its sum, its largest score (NaN: finished), what it gathered
  float* beam_top = reinterpret_cast<float*>(beam_less + a.num_beams);
  float* beam_has = beam_top + a.num_beams;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per_beam = a.parts * a.most, all = a.num_beams * per_beam;
  const uint64_t* lists = a.lists + (long long)b * all;
  for (int k = wave; k < a.num_beams; k += kMergeWaves) {
    const long long row = (long long)b * a.num_beams + k;
    const bool done = a.finished && a.finished[row];
    const float has = a.beams ? a.beams[row] : 0.f;
    float top = done ? NAN : 0.f;
    double sum = 1.0;
    if (a.normalise && !done) {
      const float first_top = lane < a.parts ? a.list_top[row * a.parts + lane] : -INFINITY;
      const double first_sum = lane < a.parts ? a.list_sum[row * a.parts + lane] : 0.0;
      top = first_top;
      for (int p = lane + 64; p < a.parts; p += 64) top = fmaxf(top, a.list_top[row * a.parts + p]);
      for (int step = 32; step > 0; step >>= 1) top = fmaxf(top, __shfl_xor(top, step));
      sum = 0.0;
      for (int p = lane; p < a.parts; p += 64) {
        const float t = p < 64 ? first_top : a.list_top[row * a.parts + p];
        const double s = p < 64 ? first_sum : a.list_sum[row * a.parts + p];
        if (t > -INFINITY) sum += t == top ? s : s * exp((double)t - (double)top);
      }
      for (int step = 32; step > 0; step >>= 1) sum += __shfl_xor(sum, step);
    }
    if (lane == 0) {
      beam_top[k] = top;
      beam_has[k] = has;
      beam_less[k] = a.normalise ? log(sum) : 0.0;
    }
  }
  if (tid == 0) filled = 0;
  uint64_t totals[HELD];  // 0: no candidate
#pragma unroll
  for (int i = 0; i < HELD; ++i) totals[i] = tid + i * kMerge < all ? lists[tid + i * kMerge] : 0;
  __syncthreads();
  uint64_t best = 0;
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    if (i * kMerge >= all) continue;
    const int c = tid + i * kMerge, k = c / per_beam;
    const uint64_t key = totals[i];
    totals[i] = 0;
    if (c < all) {
      const double has = beam_has[k], top = beam_top[k];
      double total = -INFINITY;
      if (top != top) {
        if (c == k * per_beam) total = has;
      } else if (key != 0) {
        total = key_value(key);
        total = (total == top ? 0.0 : total - top) - beam_less[k] + has;
      }
      if (total > -INFINITY) totals[i] = order_total(total);
    }
    best = totals[i] > best ? totals[i] : best;
  }
  auto key_of = [&](int c, int k) -> uint64_t { return beam_top[k] != beam_top[k] ? (uint64_t)(uint32_t)~(uint32_t)a.end : lists[c]; };

  // The num-th largest of the groups' best: of those that fewer than num are above, the smallest.
  for (int step = 1; step < 4; step <<= 1) {
    const uint64_t other = __shfl_xor(best, step);
    best = other > best ? other : best;
  }
  if ((lane & 3) == 0) group_best[tid >> 2] = best;
  __syncthreads();
  uint64_t bar, beyond = best;
  {
    int above = 0;
#pragma unroll 8
    for (int i = lane & 3; i < kGroups; i += 4) above += group_best[i] > best;
    above += __shfl_xor(above, 1);
    above += __shfl_xor(above, 2);
    bar = above < a.num ? best : ~(uint64_t)0;
    for (int step = 32; step > 0; step >>= 1) {
      const uint64_t low = __shfl_xor(bar, step), high = __shfl_xor(beyond, step);
      bar = low < bar ? low : bar;
      beyond = high > beyond ? high : beyond;
    }
    if (lane == 0) kept_total[wave] = bar, kept_key[wave] = beyond;
    __syncthreads();
    for (int w = 0; w < kMergeWaves; ++w) {
      bar = kept_total[w] < bar ? kept_total[w] : bar;
      beyond = kept_key[w] > beyond ? kept_key[w] : beyond;
    }
    beyond += 1;
  }
  if (bar == 0) bar = 1;
  // How many reach the bar: while they are many more than asked for, and not all equal, it is raised by halving.
  const int enough = a.num + kGroups;
  int count = 0;
  uint64_t probe = bar;
  for (int turn = 0;; turn ^= 1) {
    int reach = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (i * kMerge < all) reach += __popcll(__ballot(totals[i] >= probe));
    if (lane == 0) counts[turn][wave] = reach;
    __syncthreads();
    reach = 0;
    for (int w = 0; w < kMergeWaves; ++w) reach += counts[turn][w];
    if (probe == bar || reach >= a.num) {
      bar = probe;
      count = reach;
    } else {
      beyond = probe;
    }
    if (count <= enough || beyond - bar <= 1) break;
    probe = bar + (beyond - bar) / 2;
  }
  const long long out = (long long)b * a.num;
  int divisor = per_beam;  // (hidden, so that the quotients are worked out again where they are used and not kept in registers)
  asm volatile("" : "+s"(divisor));
  if (HELD * kMerge <= kKept || count <= kKept) {
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (totals[i] >= bar) {
        const int at = atomicAdd(&filled, 1), c = tid + i * kMerge, k = c / divisor;
        kept_total[at] = totals[i];
        kept_key[at] = key_of(c, k);
        kept_beam[at] = k;
      }
    __syncthreads();
    for (int first = 0; first < count; first += kGroups) {
      const int i = first + (tid >> 2);
      int rank = 0;
      uint64_t t = 0, key = 0;
      int k = 0;
      if (i < count) {
        t = kept_total[i], key = kept_key[i], k = kept_beam[i];
#pragma unroll 4
        for (int j = lane & 3; j < count; j += 4) {
          const uint64_t other = kept_total[j];
          if (other == t) rank += kept_beam[j] < k || (kept_beam[j] == k && kept_key[j] > key);
          else rank += other > t;
        }
      }
      rank += __shfl_xor(rank, 1);
      rank += __shfl_xor(rank, 2);
      if (i < count && (lane & 3) == 0 && rank < a.num) {
        a.out_totals[out + rank] = (float)total_value(t);
        a.out_parents[out + rank] = k;
        a.out_tokens[out + rank] = key_place(key);
      }
    }
    for (int i = count + tid; i < a.num; i += kMerge) {
      a.out_totals[out + i] = -INFINITY;
      a.out_parents[out + i] = a.out_tokens[out + i] = -1;
    }
    return;
  }
  // More equal totals than are held (of more candidates than are held): one after the other, each the best of those behind the last one.
  uint64_t last = ~0ull, last_key = 0;
  int last_beam = -1;
  auto before = [](uint64_t t, int k, uint64_t key, uint64_t t2, int k2, uint64_t key2) {
    return t != t2 ? t > t2 : k != k2 ? k < k2 : key > key2;
  };
  for (int n = 0; n < a.num; ++n) {
    uint64_t mine = 0, mine_key = 0;
    int mine_beam = 0;
    asm volatile("" : "+s"(divisor));
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const uint64_t t = totals[i];
      if (t < bar) continue;
      const int c = tid + i * kMerge, k = c / divisor;
      const uint64_t key = key_of(c, k);
      if (last_beam >= 0 && !before(last, last_beam, last_key, t, k, key)) continue;
      if (mine == 0 || before(t, k, key, mine, mine_beam, mine_key)) mine = t, mine_key = key, mine_beam = k;
    }
    for (int step = 1; step < 64; step <<= 1) {
      const uint64_t t = __shfl_xor(mine, step), key = __shfl_xor(mine_key, step);
      const int k = __shfl_xor(mine_beam, step);
      if (t != 0 && (mine == 0 || before(t, k, key, mine, mine_beam, mine_key))) mine = t, mine_key = key, mine_beam = k;
    }
    __syncthreads();
    if (lane == 0) kept_total[wave] = mine, kept_key[wave] = mine_key, kept_beam[wave] = mine_beam;
    __syncthreads();
    if (tid == 0) {  // (there are num of them: more than are held reach the bar)
      int w = 0;
      for (int o = 1; o < kMergeWaves; ++o)
        if (kept_total[o] != 0 && (kept_total[w] == 0 || before(kept_total[o], kept_beam[o], kept_key[o], kept_total[w], kept_beam[w], kept_key[w]))) w = o;
      first_best = w;
      a.out_totals[out + n] = (float)total_value(kept_total[w]);
      a.out_parents[out + n] = kept_beam[w];
      a.out_tokens[out + n] = key_place(kept_key[w]);
    }
    __syncthreads();
    last = kept_total[first_best];
    last_key = kept_key[first_best];
    last_beam = kept_beam[first_best];
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

// Bound by memory: every state is read and written once, four accesses of a thread in flight.  Four arrays of 32 x 8 states of
// 128 KB (134 MB written, what several picked is read once): 28 us.
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

// How a selection is spread: as many workgroups a row as the machine holds at once (six on a CU: one more would be a second round)
// and as the last step can hold candidates of.  Of a row of 1 000 000 float32 scores (the best ten) 16, 64 and 256
// workgroups take 30, 22 and 19 us.
constexpr int kResident = 6 * 256, kMostParts = 256;
struct SelectPlan {
  int parts, each;
};
static SelectPlan select_plan(int num_batch, int num_beams, int num_values, int num) {
  const long long rows = (long long)num_batch * num_beams;
  const int tiles = (num_values + kThreads * kEach - 1) / (kThreads * kEach), most = std::min(num, num_values);
  const int wanted = (int)std::max<long long>(1, std::min<long long>({kResident / rows, kMostParts, kMostCandidates / ((long long)num_beams * most)}));
  SelectPlan p;
  p.each = (tiles + wanted - 1) / wanted;
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
  return (long long)SelectScratch(nullptr, (long long)num_batch * num_beams, select_plan(num_batch, num_beams, num_values, num).parts,
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
    const SelectPlan p = select_plan(num_batch, num_beams, num_values, num);
    const long long rows = (long long)num_batch * num_beams;
    const SelectScratch w(workspace, rows, p.parts, std::min(num, num_values));
    want(workspace && workspace_bytes >= (long long)w.bytes, "select: the workspace is too small");
    SelectArgs a{scores, stride_b, stride_k, num_batch, num_beams, num_values, beams, finished, normalise, end, num,
                 out_totals, out_parents, out_tokens, p.parts, p.each, std::min(num, num_values), w.lists, w.tops, w.sums};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int candidates = num_beams * p.parts * a.most;
    // (a launch has fewer than 2^32 threads; what is left goes through the same workspace behind it)
    const long long step = std::min<long long>(0xffffffffll / kMerge, 0xffffffffll / kThreads / ((long long)num_beams * p.parts));
    for (long long first = 0; first < num_batch; first += step) {
      a.num_batch = (int)std::min<long long>(step, num_batch - first);
      a.scores = static_cast<const unsigned char*>(scores) + first * stride_b * element_size(type);
      a.beams = beams ? beams + first * num_beams : nullptr;
      a.finished = finished ? finished + first * num_beams : nullptr;
      a.out_totals = out_totals + first * num;
      a.out_parents = out_parents + first * num;
      a.out_tokens = out_tokens + first * num;
      with_type(type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const dim3 grid((unsigned)a.num_batch * num_beams * p.parts);
        if (normalise) hipLaunchKernelGGL((select_part_kernel<T, true>), grid, dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((select_part_kernel<T, false>), grid, dim3(kThreads), 0, s, a);
      });
      const dim3 grid((unsigned)a.num_batch);
      if (candidates <= 2 * kMerge) hipLaunchKernelGGL(select_merge_kernel<2>, grid, dim3(kMerge), (size_t)num_beams * 16, s, a);
      else hipLaunchKernelGGL(select_merge_kernel<kMostCandidates / kMerge>, grid, dim3(kMerge), (size_t)num_beams * 16, s, a);
    }
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
