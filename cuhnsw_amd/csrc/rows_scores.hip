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
  const int groups = (a.num_dims + a.group - 1) / a.group;
  const long long step = std::max<long long>(1, (1ll << 31) / lanes), width = ((long long)a.num_dims + 31) / 32 * 16;  // (a launch has fewer than 2^32 threads)
  with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    for (long long first = 0; first < a.num_rows; first += step) {
      const long long rows = std::min(step, a.num_rows - first);
      uint16_t *scales = static_cast<uint16_t*>(a.scales) + first * groups, *offsets = static_cast<uint16_t*>(a.offsets);
      hipLaunchKernelGGL(pack_kernel<T>, dim3((unsigned)((rows * lanes + 255) / 256)), dim3(256), 0, stream,
                         static_cast<const T*>(a.rows) + first * a.row_stride, a.row_stride, rows, a.num_dims, a.group, lanes,
                         a.codes + first * width, scales, offsets ? offsets + first * groups : nullptr, a.scale_type == TYPE_BF16);
    }
  });
  HIP_CHECK(hipGetLastError());
}

// ----------------------------------------------------------------------------------------------- products
// On the matrix cores, in float16: a code less 8 (or the code) is exact there, and so is a query as one or two planes of
// float16, once a power of two has brought its largest element to [2^14, 2^15): a float32 is the sum of its rounding to 11 bits
// and the rounding of the rest (off by 2^-23 of it, or by 2^-39 of the largest element where that is more), a bfloat16 or a
// float16 is one plane.  Products are summed in 32 bits per group of elements; the group's scale is applied to that sum, so
// no weight is ever rounded.  Offsets meet the group's sum of query elements.
//
// Queries are laid out as the lanes want them: for a tile of 16 queries and a unit of 32 elements, 16 bytes for every quarter of the
// unit and query.  That is a launch of its own (prepare_kernel), or, of one or two, every workgroup's first step, into its LDS.
constexpr int kManyWaves = 4;      // wavefronts of a workgroup for many queries
constexpr int kManyResident = 768;  // such workgroups at work at a time, as the plan counts: three on a CU (the instances' registers and LDS
                                    // let it hold two to six: two with float32 queries, four tiles and chunks of four units)
constexpr int kTile = 16, kUnit = 32, kRowTiles = 4;  // queries or rows of a matrix product, elements of it; row tiles of a wavefront

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bfloat2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef float float4_t __attribute__((ext_vector_type(4)));

struct ScoresArgs {
  const unsigned char* codes;
  const uint16_t *scales, *offsets;
  int scale_bf16;
  int num_rows, num_dims, group;
  int units, groups;  // of a row
  const void* queries;
  long long query_stride;
  int num_queries;
  float alpha;
  const float* bias;
  void* out;
  int out_type;
  long long out_stride;
  int padded_units;        // units that the planes hold: the last are zero
  _Float16* planes;        // [planes][query tile][unit][quarter][16][8]
  size_t plane;            // elements of one plane
  signed char* exponents;  // of every query: what its scores are to be scaled by
  float* sums;             // [query tile][group][16]: sums of the groups' elements
  int query_blocks, row_blocks, split, blocks_each;
};

// Eight elements of a query, 0 behind the last one.
template <typename T>
__device__ inline LoosePack<T, 8> eight_of(const T* q, int first, int num_dims) {
  LoosePack<T, 8> x;
  if (first + 8 <= num_dims) {
    x = *reinterpret_cast<const LoosePack<T, 8>*>(q + first);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x.at[e] = first + e < num_dims ? q[first + e] : narrow<T>(0.f);
  }
  return x;
}

// A workgroup lays a query out.  A power of two takes its largest magnitude to [2^14, 2^15) (a float16 query stays as it is, and
// one that is zero or not finite too): returned is the exponent of the largest element.  put(w, high, low) gets the planes of elements
// 8 w to 8 w + 7, in the order in which the codes of a word come apart (0 4 1 5 2 6 3 7), put_sum(g, sum) the sums of the
// groups if `with_sums`.
template <typename T, typename Put, typename PutSum>
__device__ inline int lay_out(const T* q, int num_dims, int pieces, int group, int groups, bool with_sums, float* per_wave, Put put, PutSum put_sum) {
  const int tid = threadIdx.x, threads = blockDim.x, lanes = group / 8;
  const LoosePack<T, 8> held = eight_of(q, tid * 8, num_dims);
  int exponent = 14;
  if (!std::is_same_v<T, _Float16>) {
    float most = 0.f;
    auto look_at = [&](const LoosePack<T, 8>& x) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = fabsf(widen(x.at[e]));
        most = y < INFINITY ? fmaxf(most, y) : INFINITY;  // (a NaN too)
      }
    };
    look_at(held);
    for (int w = tid + threads; w * 8 < num_dims; w += threads) look_at(eight_of(q, w * 8, num_dims));
    for (int step = 32; step > 0; step >>= 1) most = fmaxf(most, __shfl_xor(most, step));
    if ((tid & 63) == 0) per_wave[tid >> 6] = most;
    __syncthreads();
    for (int w = 0; w < threads / 64; ++w) most = fmaxf(most, per_wave[w]);
    __syncthreads();
    if (most > 0.f && most < INFINITY) exponent = max(ilogbf(most), -126);  // (a byte holds it)
  }
  for (int first = 0; first < pieces; first += threads) {  // (lanes of one group come this way together)
    const int w = first + tid;
    const LoosePack<T, 8> x = first == 0 ? held : eight_of(q, w * 8, num_dims);
    half8_t high, low;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = ldexpf(widen(x.at[(e & 1) * 4 + (e >> 1)]), 14 - exponent);
      high[e] = (_Float16)y;
      low[e] = (_Float16)(y - (float)high[e]);
      sum += ldexpf(y, -14);
    }
    if (w < pieces) put(w, high, low);
    if (with_sums) {
      for (int step = 1; step < lanes; step <<= 1) sum += __shfl_xor(sum, step);
      if (w % lanes == 0 && w / lanes < groups) put_sum(w / lanes, sum);
    }
  }
  return exponent;
}

template <typename T>
__global__ void __launch_bounds__(256) prepare_kernel(ScoresArgs a, int planes) {
  __shared__ float per_wave[4];
  const int m = blockIdx.x, tile = m / kTile, i = m % kTile;
  const bool there = m < a.num_queries;  // (the last tile is filled up with zeros)
  const T* q = static_cast<const T*>(a.queries) + (there ? m : 0) * a.query_stride;
  _Float16* to = a.planes + (size_t)tile * kTile * a.padded_units * kUnit;
  const int exponent = lay_out(
      q, there ? a.num_dims : 0, a.padded_units * 4, a.group, a.groups, a.offsets != nullptr, per_wave,
      [&](int w, half8_t high, half8_t low) {
        *reinterpret_cast<half8_t*>(to + ((size_t)w * kTile + i) * 8) = high;
        if (planes == 2) *reinterpret_cast<half8_t*>(to + a.plane + ((size_t)w * kTile + i) * 8) = low;
      },
      [&](int g, float sum) { a.sums[((size_t)tile * a.groups + g) * kTile + i] = sum; });
  if (threadIdx.x == 0) a.exponents[m] = (signed char)exponent;
}

// The eight codes of a word, less 8 or as they are, as float16, in the order 0 4 1 5 2 6 3 7: a code behind the exponent of 1024
// is 1024 more (16 times the code behind it for every other one), and what is too much goes off exactly (the well-known way to
// small whole numbers in floating point, by the exponent below which their bits lie).
template <bool CENTRED>
__device__ inline half8_t codes_of(uint32_t word) {
  constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;
  uint32_t k1024 = 0x64006400u;
  asm("" : "+v"(k1024));  // (in a vector register: one instruction takes the bits out and puts the exponent in)
  const half2_t low = CENTRED ? half2_t{-1032.f16, -1032.f16} : half2_t{-1024.f16, -1024.f16};
  const half2_t high = CENTRED ? half2_t{-72.f16, -72.f16} : half2_t{-64.f16, -64.f16}, sixteenth = {0.0625f16, 0.0625f16};
  const uint32_t next = word >> 8;
  const half2_t a = __builtin_bit_cast(half2_t, (word & kLow) | k1024) + low;
  const half2_t b = __builtin_elementwise_fma(__builtin_bit_cast(half2_t, (word & kHigh) | k1024), sixteenth, high);
  const half2_t c = __builtin_bit_cast(half2_t, (next & kLow) | k1024) + low;
  const half2_t d = __builtin_elementwise_fma(__builtin_bit_cast(half2_t, (next & kHigh) | k1024), sixteenth, high);
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Scales or offsets of a chunk's N groups, two in a word.
typedef uint32_t loose32 __attribute__((aligned(2)));
typedef uint64_t loose64 __attribute__((aligned(2)));
template <int N>
struct Groups {
  uint32_t words[(N + 1) / 2];
  __device__ uint16_t operator[](int g) const { return (uint16_t)(words[g / 2] >> (g % 2 * 16)); }
};
// from group `first` on, at once where they are all the row's own (the others are not looked at)
template <int N>
__device__ inline Groups<N> load_groups(const uint16_t* row, int first, int groups) {
  Groups<N> x;
  const uint16_t* from = row + first;
  if (first + N <= groups) {
    if constexpr (N == 1) {
      x.words[0] = from[0];
    } else if constexpr (N == 2) {
      x.words[0] = *reinterpret_cast<const loose32*>(from);
    } else if constexpr (N == 3) {
      x.words[0] = *reinterpret_cast<const loose32*>(from);
      x.words[1] = from[2];
    } else {
      const uint64_t both = *reinterpret_cast<const loose64*>(from);
      x.words[0] = (uint32_t)both;
      x.words[1] = (uint32_t)(both >> 32);
    }
  } else {
    for (int w = 0; w < (N + 1) / 2; ++w)
      x.words[w] = (uint32_t)row[min(first + 2 * w, groups - 1)] | (uint32_t)row[min(first + 2 * w + 1, groups - 1)] << 16;
  }
  return x;
}
// of every quarter of the wavefront its word, to all lanes
__device__ inline void from_quarters(uint32_t word, uint32_t (&all)[4]) {
  const auto halves = __builtin_amdgcn_permlane32_swap(word, word, false, false);
  const auto low = __builtin_amdgcn_permlane16_swap(halves[0], halves[0], false, false);
  const auto high = __builtin_amdgcn_permlane16_swap(halves[1], halves[1], false, false);
  all[0] = low[0];
  all[1] = low[1];
  all[2] = high[0];
  all[3] = high[1];
}
template <int N>
__device__ inline void from_quarters(const Groups<N>& x, Groups<N> (&all)[4]) {
#pragma unroll
  for (int w = 0; w < (N + 1) / 2; ++w) {
    uint32_t words[4];
    from_quarters(x.words[w], words);
#pragma unroll
    for (int q = 0; q < 4; ++q) all[q].words[w] = words[q];
  }
}

// the four words of a unit's codes in each of four slots, quarter by quarter of the wavefront -> the quarters' own words of
// each slot
__device__ inline void exchange(uint4 words, uint32_t (&slots)[4]) {
  const auto ac = __builtin_amdgcn_permlane32_swap(words.x, words.z, false, false);
  const auto bd = __builtin_amdgcn_permlane32_swap(words.y, words.w, false, false);
  const auto lo = __builtin_amdgcn_permlane16_swap(ac[0], bd[0], false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(ac[1], bd[1], false, false);
  slots[0] = lo[0];
  slots[1] = lo[1];
  slots[2] = hi[0];
  slots[3] = hi[1];
}

// Among four neighbouring lanes: of lane l, x[0..3] are row 0..3 of its column; afterwards they are column 0..3 of row l.
__device__ inline void transpose_quad(uint32_t (&x)[4]) {
  const int l = threadIdx.x & 3;
  auto swap = [&](uint32_t& low, uint32_t& high, bool upper, auto dpp) {
    const uint32_t their_low = dpp(low), their_high = dpp(high);
    low = upper ? their_high : low;
    high = upper ? high : their_low;
  };
  auto next = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xB1, 0xf, 0xf, true); };     // lanes 1 0 3 2
  auto over = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4E, 0xf, 0xf, true); };     // lanes 2 3 0 1
  swap(x[0], x[1], l & 1, next);
  swap(x[2], x[3], l & 1, next);
  swap(x[0], x[2], l & 2, over);
  swap(x[1], x[3], l & 2, over);
}

// A lane's scores: RT rows one after the other from `row` on, for four queries of every tile, whose exponents are the bytes of
// a word.  Where a score is two bytes four neighbouring lanes exchange theirs first: each then has all of their rows for one of
// the four queries, and stores 16 bytes at a time.
template <int RT, int MT>
__device__ inline void store_scores(const ScoresArgs& a, const float4_t (&acc)[RT][MT], int tile0, int c, long long row, const uint32_t (&exponents)[MT],
                                    const float (&bias)[RT]) {
  const int l = threadIdx.x & 3;
  float y[MT][4][RT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int exponent = (signed char)(exponents[m] >> (8 * r));
#pragma unroll
      for (int t = 0; t < RT; ++t) y[m][r][t] = fmaf(a.alpha, ldexpf(acc[t][m][r], exponent), bias[t]);
    }
  if (a.out_type == TYPE_F32) {
    const int rows = (int)max(0ll, min((long long)RT, a.num_rows - row));
    float* to = static_cast<float*>(a.out) + (tile0 * kTile + c * 4) * a.out_stride + row;
#pragma unroll
    for (int m = 0; m < MT; ++m, to += kTile * a.out_stride)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        LoosePack<float, RT> together;
#pragma unroll
        for (int t = 0; t < RT; ++t) together.at[t] = y[m][r][t];
        if ((tile0 + m) * kTile + c * 4 + r < a.num_queries) {
          if (rows == RT) {
            *reinterpret_cast<LoosePack<float, RT>*>(to + r * a.out_stride) = together;
          } else {
#pragma unroll
            for (int t = 0; t < RT; ++t)
              if (t < rows) to[r * a.out_stride + t] = together.at[t];
          }
        }
      }
    return;
  }
  uint32_t words[MT][RT / 2][4];  // two rows in a word
  auto round_all = [&](auto* two) {
    using Two = std::remove_pointer_t<decltype(two)>;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int w = 0; w < RT / 2; ++w)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          words[m][w][r] = __builtin_bit_cast(uint32_t, __builtin_convertvector((float2_t{y[m][r][2 * w], y[m][r][2 * w + 1]}), Two));
  };
  if (a.out_type == TYPE_BF16) round_all(static_cast<bfloat2_t*>(nullptr));
  else round_all(static_cast<half2_t*>(nullptr));
  const long long first = row - l * RT;  // of the four lanes' rows
  const int rows = (int)max(0ll, min(4ll * RT, a.num_rows - first));
  uint16_t* to = static_cast<uint16_t*>(a.out) + (tile0 * kTile + c * 4 + l) * a.out_stride + first;
#pragma unroll
  for (int m = 0; m < MT; ++m, to += kTile * a.out_stride) {
#pragma unroll
    for (int w = 0; w < RT / 2; ++w) transpose_quad(words[m][w]);
    if ((tile0 + m) * kTile + c * 4 + l >= a.num_queries) continue;
    if (rows == 4 * RT) {
#pragma unroll
      for (int i = 0; i < RT / 2; ++i) {
        struct __attribute__((packed, aligned(2))) Loose128 {
          uint32_t at[4];
        } eight;
#pragma unroll
        for (int e = 0; e < 4; ++e) eight.at[e] = words[m][(i * 4 + e) % (RT / 2)][(i * 4 + e) / (RT / 2)];
        *reinterpret_cast<Loose128*>(to + i * 8) = eight;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4 * RT; ++i)
        if (i < rows) to[i] = (uint16_t)(words[m][i / 2 % (RT / 2)][i / 2 / (RT / 2)] >> (i % 2 * 16));
    }
  }
}
// the exponents of queries c * 4 to c * 4 + 3 of a tile
__device__ inline uint32_t exponents_at(const signed char* of_tile, int c) { return *reinterpret_cast<const uint32_t*>(of_tile + c * 4); }
template <int RT>
__device__ inline void bias_at(const ScoresArgs& a, long long row, float (&bias)[RT]) {
#pragma unroll
  for (int t = 0; t < RT; ++t) bias[t] = a.bias && row + t < a.num_rows ? a.bias[row + t] : 0.f;
}

// Few queries: bound by the rows' codes (one query: 1 000 000 x 512 57 us, 4.8 TB/s; 16 384 x 4096 12 us, 3.1 TB/s, of
// which the launch and the layout of the query are 4).  A wavefront has 64 rows (four tiles of 16) and one tile of queries, and goes over the
// elements in chunks of UC units, two chunks ahead; `split` wavefronts of the workgroup share the chunks of the same rows.
// Rows 4 j to 4 j + 3 are lane j's in the four tiles, so that it stores them together.
// A load of 16 bytes brings a unit's codes to a lane: four such slots, one for each quarter of the wavefront, are
// different units of one row tile, or on short rows of several.  Four lane exchanges then give every quarter its quarter
// of each slot, so one matrix product covers one unit, inside one group.
// OWN: the workgroup lays the queries out itself (at most 16), else T is not looked at.
template <typename T, int UC, int GU, int PLANES, bool CENTRED, bool OWN>
__global__ void __launch_bounds__(512) scores_few_kernel(ScoresArgs a) {
  constexpr int kGroups = (UC + GU - 1) / GU;  // of a chunk
  extern __shared__ __align__(16) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int j = lane & 15, c = lane >> 4;
  const int per_block = waves / a.split, block = blockIdx.x / a.query_blocks, tile = blockIdx.x % a.query_blocks;
  const int share = wave % a.split, in_block = wave / a.split;
  const long long row0 = ((long long)block * per_block + in_block) * (kRowTiles * kTile), last_row = a.num_rows - 1;
  const int chunks = (a.units + UC - 1) / UC, per_share = (chunks + a.split - 1) / a.split;
  const int chunk0 = share * per_share, chunk1 = row0 <= last_row ? min(chunks, chunk0 + per_share) : 0;

  struct Stage {
    uint4 words[UC];
    Groups<kGroups> scales, offsets;  // of row tile c's row of the lane
    half8_t query[UC][PLANES];
  };
  const unsigned char* from[UC];
  int unit_of[UC];
#pragma unroll
  for (int i = 0; i < UC; ++i) {
    const int slot = 4 * i + c;
    unit_of[i] = slot % UC;
    from[i] = a.codes + min(row0 + j * kRowTiles + slot / UC, last_row) * ((long long)a.units * 16);
  }
  const long long groups_of = min(row0 + j * kRowTiles + c, last_row) * a.groups;
  const _Float16* planes = a.planes + (size_t)tile * kTile * a.padded_units * kUnit + lane * 8;
  auto load = [&](Stage& s, int chunk) {
    if (chunk >= chunk1) return;
#pragma unroll
    for (int i = 0; i < UC; ++i) s.words[i] = *reinterpret_cast<const uint4*>(from[i] + min(chunk * UC + unit_of[i], a.units - 1) * 16);
    s.scales = load_groups<kGroups>(a.scales + groups_of, chunk * UC / GU, a.groups);
    if (!CENTRED) s.offsets = load_groups<kGroups>(a.offsets + groups_of, chunk * UC / GU, a.groups);
    if (!OWN)
#pragma unroll
      for (int u = 0; u < UC; ++u)
#pragma unroll
        for (int p = 0; p < PLANES; ++p) s.query[u][p] = *reinterpret_cast<const half8_t*>(planes + p * a.plane + (size_t)(chunk * UC + u) * 512);
  };
  Stage even, odd;
  load(even, chunk0);
  load(odd, chunk0 + 1);

  // (own queries) [planes][unit][quarter][query][8], then the groups' sums [group][16], then the exponents
  const int own_queries = min(kTile, a.num_queries), own_plane = a.padded_units * kUnit * own_queries;
  _Float16* own = reinterpret_cast<_Float16*>(lds);
  float* own_sums = reinterpret_cast<float*>(own + (size_t)PLANES * own_plane);
  signed char* own_exponents = reinterpret_cast<signed char*>(own_sums + (CENTRED ? 0 : kTile * a.groups));
  float* per_wave = reinterpret_cast<float*>(own_exponents + kTile);
  float4_t* partial = reinterpret_cast<float4_t*>(OWN ? reinterpret_cast<unsigned char*>(per_wave + 8) : lds);
  if (OWN) {
    for (int i = 0; i < own_queries; ++i) {
      const T* q = static_cast<const T*>(a.queries) + i * a.query_stride;
      const int exponent = lay_out(
          q, a.num_dims, a.padded_units * 4, a.group, a.groups, !CENTRED, per_wave,
          [&](int w, half8_t high, half8_t low) {
            *reinterpret_cast<half8_t*>(own + ((size_t)w * own_queries + i) * 8) = high;
            if (PLANES == 2) *reinterpret_cast<half8_t*>(own + own_plane + ((size_t)w * own_queries + i) * 8) = low;
          },
          [&](int g, float sum) { own_sums[g * kTile + i] = sum; });
      if (threadIdx.x == 0) own_exponents[i] = (signed char)exponent;
    }
    __syncthreads();
  }

  float4_t acc[kRowTiles][1];
#pragma unroll
  for (int t = 0; t < kRowTiles; ++t) acc[t][0] = float4_t{0.f, 0.f, 0.f, 0.f};
  auto use = [&](const Stage& s, int chunk) {
    half8_t query[UC][PLANES];
#pragma unroll
    for (int u = 0; u < UC; ++u)
#pragma unroll
      for (int p = 0; p < PLANES; ++p)
        query[u][p] = OWN ? *reinterpret_cast<const half8_t*>(own + p * own_plane + (((chunk * UC + u) * 4 + c) * own_queries + min(j, own_queries - 1)) * 8)
                          : s.query[u][p];
    Groups<kGroups> scales[kRowTiles], offsets[kRowTiles];
    from_quarters(s.scales, scales);
    if (!CENTRED) from_quarters(s.offsets, offsets);
    float4_t temp;
#pragma unroll
    for (int i = 0; i < UC; ++i) {
      uint32_t slots[4];
      exchange(s.words[i], slots);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int slot = 4 * i + q, t = slot / UC, u = slot % UC;
        const half8_t codes = codes_of<CENTRED>(slots[q]);
        if (u % GU == 0) temp = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = PLANES - 1; p >= 0; --p) temp = __builtin_amdgcn_mfma_f32_16x16x32_f16(query[u][p], codes, temp, 0, 0, 0);
        if (u % GU != GU - 1 && u != UC - 1) continue;
        const float scale = half_bits(scales[t][u / GU], a.scale_bf16) * 0x1p-14f;
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[t][0][r] = fmaf(scale, temp[r], acc[t][0][r]);
        if (!CENTRED) {  // (behind the last group there is nothing)
          const int group = chunk * UC / GU + u / GU, held = min(group, a.groups - 1);
          const float* sums = OWN ? own_sums + held * kTile : a.sums + ((size_t)tile * a.groups + held) * kTile;
          const float4_t x = *reinterpret_cast<const float4_t*>(sums + c * 4);
          const float offset = group == held ? half_bits(offsets[t][u / GU], a.scale_bf16) : 0.f;
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[t][0][r] = fmaf(offset, x[r], acc[t][0][r]);
        }
      }
    }
  };
  for (int chunk = chunk0; chunk < chunk1; chunk += 2) {
    use(even, chunk);
    load(even, chunk + 2);
    if (chunk + 1 < chunk1) {
      use(odd, chunk + 1);
      load(odd, chunk + 3);
    }
  }
  if (a.split > 1) {
    if (share > 0)
#pragma unroll
      for (int t = 0; t < kRowTiles; ++t) partial[(((share - 1) * per_block + in_block) * kRowTiles + t) * 64 + lane] = acc[t][0];
    __syncthreads();
    if (share > 0) return;
    for (int s = 0; s < a.split - 1; ++s)
#pragma unroll
      for (int t = 0; t < kRowTiles; ++t) acc[t][0] += partial[((s * per_block + in_block) * kRowTiles + t) * 64 + lane];
  }
  const uint32_t exponents[1] = {exponents_at(OWN ? own_exponents : a.exponents + tile * kTile, c)};
  float bias[kRowTiles];
  bias_at(a, row0 + j * kRowTiles, bias);
  store_scores<kRowTiles, 1>(a, acc, tile, c, row0 + j * kRowTiles, exponents, bias);
}

// Many queries: a workgroup of kManyWaves wavefronts has 32 rows for each of them, and goes over `blocks_each` blocks of MT
// tiles of queries, chunk by chunk of UC units.  The queries' planes of a chunk go through LDS (straight from memory, the
// next chunk's while this one is at work), so the wavefronts share what they read of them; a unit's planes stay in
// registers over the wavefront's two row tiles.  Rows 2 j and 2 j + 1 are lane j's in the two tiles, so that it stores them
// together.
//
// What bounds it: instructions of the vector units.  For every matrix product of 16 x 16 x 32 a quarter of a word comes apart
// and four sums are scaled (four more with offsets).  131 072 x 1024 by 1024 bfloat16 queries: 371 us, 741 TFLOP/s (a library's product
// in float16 reaches 1128 here); 200 003 x 960 by 33 float32 queries with offsets (two planes): 74 us, of which vector instructions 38 and
// matrix products 16; 500 000 x 128 by 256 with offsets: 107 us, 68 of them without
// the stores of its 256 MB of scores, which the next block's work hides little of: a wavefront waits for them before it uses what was
// brought meanwhile.
//
// Workgroups of 4, 6 and 8 wavefronts take 80, 116, 105 us for the second, 384, 583, 478 for the first; registers for four
// workgroups on a CU instead of three spill, 84 and 556.
template <int UC, int GU, int MT, int PLANES, bool CENTRED>
__global__ void __launch_bounds__(64 * kManyWaves, 3) scores_many_kernel(ScoresArgs a) {
  constexpr int RT = 2, kLoads = UC * RT / 4;
  constexpr int kGroups = (UC + GU - 1) / GU, kPieces = UC * MT * PLANES;  // pieces of 1 KB: what a wavefront reads at once
  __shared__ half8_t queries[2][kPieces][64];
  __shared__ float4_t sums[CENTRED ? 1 : 2][CENTRED ? 1 : MT][16];  // [..][group of the chunk * 4 + quarter]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, c = lane >> 4;
  // workgroups of the same rows one after the other on the same chiplet, whose L2 then holds the rows
  const int shares = (a.query_blocks + a.blocks_each - 1) / a.blocks_each, turn = blockIdx.x >> 3;
  const int block = (turn / shares) * 8 + (blockIdx.x & 7), query_block0 = (turn % shares) * a.blocks_each;
  if (block >= a.row_blocks) return;
  const int last_tile = (a.num_queries - 1) / kTile, chunks = (a.units + UC - 1) / UC;
  const long long row0 = (long long)block * (kManyWaves * RT * kTile) + wave * (RT * kTile), last_row = a.num_rows - 1;

  const unsigned char* from[kLoads];
  int unit_of[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int slot = 4 * i + c;
    unit_of[i] = slot % UC;
    from[i] = a.codes + min(row0 + j * RT + slot / UC, last_row) * ((long long)a.units * 16);
  }
  // (an even quarter has the first row tile's scales and offsets, an odd one the second's; offsets come to the upper half)
  const uint16_t* groups_of = (CENTRED || c < 2 ? a.scales : a.offsets) + min(row0 + j * RT + (c & 1), last_row) * a.groups;
  uint4 words[kLoads];
  Groups<kGroups> held;
  auto load = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) words[i] = *reinterpret_cast<const uint4*>(from[i] + min(chunk * UC + unit_of[i], a.units - 1) * 16);
    held = load_groups<kGroups>(groups_of, chunk * UC / GU, a.groups);
  };
  // piece (u, m, p) of a chunk: 64 x 16 bytes that lie in a row in the planes
  auto bring = [&](int query_block, int chunk, int buffer) {
    for (int piece = wave; piece < kPieces; piece += kManyWaves) {
      const int p = piece % PLANES, m = piece / PLANES % MT, u = piece / PLANES / MT, tile = min(query_block * MT + m, last_tile);
      const _Float16* there = a.planes + p * a.plane + ((size_t)tile * a.padded_units + chunk * UC + u) * (kTile * kUnit) + lane * 8;
      __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(there)),
                                       (__attribute__((address_space(3))) void*)&queries[buffer][piece][0], 16, 0, 0);
    }
    if (!CENTRED && wave < MT) {  // the sums of the chunk's groups, a float for each lane
      const size_t tile = min(query_block * MT + wave, last_tile);
      // (behind the row's last group the query's own sum of that one: it meets an offset of 0, and 0 times what is not finite is not 0)
      const int at = min(chunk * UC / GU + lane / kTile, a.groups - 1) * kTile + lane % kTile;
      __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(a.sums + tile * a.groups * kTile + at)),
                                       (__attribute__((address_space(3))) void*)&sums[buffer][wave][0], 4, 0, 0);
    }
  };
  const int query_blocks = min(a.blocks_each, a.query_blocks - query_block0);
  float4_t acc[RT][MT];
  uint32_t exponents[MT];
  float bias[RT];
  bias_at(a, row0 + j * RT, bias);
  int query_block = query_block0, chunk = 0;
  bring(query_block, 0, 0);
  load(0);
  for (int step = 0;; ++step) {
    // What was brought is in LDS once every wavefront has waited for its own loads.  A block's scores are stored behind that wait:
    // they have the next chunk's work to get there.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const int buffer = step & 1;
    if (chunk == 0) {
      if (step > 0) store_scores<RT, MT>(a, acc, (query_block - 1) * MT, c, row0 + j * RT, exponents, bias);
      if (query_block == query_block0 + query_blocks) break;
#pragma unroll
      for (int m = 0; m < MT; ++m) exponents[m] = exponents_at(a.exponents + min(query_block * MT + m, last_tile) * kTile, c);
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    {
      uint32_t word[RT][UC];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        uint32_t slots[4];
        exchange(words[i], slots);
#pragma unroll
        for (int q = 0; q < 4; ++q) word[(4 * i + q) / UC][(4 * i + q) % UC] = slots[q];
      }
      Groups<kGroups> quarters[4];
      from_quarters(held, quarters);
      float scale[RT][kGroups], offset[RT][kGroups];
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          scale[t][g] = half_bits(quarters[t][g], a.scale_bf16) * 0x1p-14f;
          // (behind the last group there is nothing)
          offset[t][g] = CENTRED || chunk * UC / GU + g >= a.groups ? 0.f : half_bits(quarters[2 + t][g], a.scale_bf16);
        }
      if (++chunk == chunks) {
        chunk = 0;
        ++query_block;
      }
      if (query_block < query_block0 + query_blocks) {
        bring(query_block, chunk, buffer ^ 1);
        load(chunk);
      }
      float4_t temp[RT][MT];
#pragma unroll
      for (int u = 0; u < UC; ++u) {
        half8_t query[MT][PLANES];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int p = 0; p < PLANES; ++p) query[m][p] = queries[buffer][(u * MT + m) * PLANES + p][lane];
        float4_t x[MT];
        if (!CENTRED && (u % GU == GU - 1 || u == UC - 1))
#pragma unroll
          for (int m = 0; m < MT; ++m) x[m] = sums[buffer][m][u / GU * 4 + c];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const half8_t codes = codes_of<CENTRED>(word[t][u]);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if (u % GU == 0) temp[t][m] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = PLANES - 1; p >= 0; --p) temp[t][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(query[m][p], codes, temp[t][m], 0, 0, 0);
          }
        }
        if (u % GU != GU - 1 && u != UC - 1) continue;
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              acc[t][m][r] = fmaf(scale[t][u / GU], temp[t][m][r], acc[t][m][r]);
              if (!CENTRED) acc[t][m][r] = fmaf(offset[t][u / GU], x[m][r], acc[t][m][r]);
            }
      }
    }
  }
}

inline int units_of(int num_dims) { return (num_dims + kUnit - 1) / kUnit; }
inline int planes_of(int query_type) { return query_type == TYPE_F32 ? 2 : 1; }

// How a call is spread.  Times in us, both sides of each rule:
//
// Many queries' kernel from 384 pairs of a workgroup's rows (128) and a query tile (16) on, where it fills the machine.  16 384 x 1024
// bf16: 17 queries (256 pairs) 10.4 few, 11.9 many; 33 (384): 13.3, 13.2; 64: 15.2, 13.6; 256: 32.0, 19.0.  16 384 x 960 fp32, 33
// queries: 18.3, 16.4.  32 000 x 128 fp16, 17 queries (500): 6.4, 5.9.
//
// One or two queries are laid out by every workgroup, more by a launch of their own.  100 000 x 50 fp32: 1 query 4.7 and 6.4, 4 queries
// 8.4 and 7.2; 131 072 x 1024 bf16: 19.8 and 22.7, 25.9 and 22.7.
//
// Wavefronts that share a row's elements: doubled while the rows make fewer than 4096 of them (four on a SIMD).  One bf16 query, 16 384 x
// 4096: one 28.7, eight 11.9; 65 536 x 4096: one 37.2, four 32.4, eight 43.0; 262 144 x 1024: one 30.6, eight 73.1.
struct ScoresPlan {
  int chunk, padded_units, planes, groups;  // units of a chunk; of a row, with the units that fill the last chunk up
  int query_tiles;                          // of a workgroup; 0: few queries
  bool own;                                 // few queries, laid out by the workgroups themselves
  int split, waves, query_blocks, row_blocks;
  int blocks_each;                          // many queries: blocks of them that a workgroup goes over
  size_t lds;
  ScoresPlan(long long num_rows, int num_dims, int group, int query_type, int num_queries) {
    const int units = units_of(num_dims), tiles = (num_queries + kTile - 1) / kTile;
    planes = planes_of(query_type);
    groups = (num_dims + group - 1) / group;
    query_blocks = (tiles + 3) / 4;
    const long long blocks = (num_rows + kManyWaves * 32 - 1) / (kManyWaves * 32);
    query_tiles = tiles > 1 && blocks * tiles >= 384 ? (tiles + query_blocks - 1) / query_blocks : 0;
    own = false;
    lds = 0;
    blocks_each = 1;
    if (query_tiles) {
      chunk = units <= 2 ? 2 : 4;
      split = 1;
      waves = kManyWaves;
      row_blocks = (int)blocks;
      // into how many workgroups the query blocks of the same rows are divided: rounds of workgroups times the chunks of each,
      // and the loads that nothing hides at its beginning
      const int chunks = (units + chunk - 1) / chunk;
      long long least = 0;
      for (int shares = 1; shares <= std::min(query_blocks, 16); ++shares) {
        const int each = (query_blocks + shares - 1) / shares;
        const long long time = (blocks * ((query_blocks + each - 1) / each) + kManyResident - 1) / kManyResident * ((long long)each * chunks + 2);
        if (shares == 1 || time < least) least = time, blocks_each = each;
      }
    } else {
      chunk = std::min(units, 4);
      query_blocks = tiles;
      const long long row_waves = (num_rows + 63) / 64;
      const int chunks = (units + chunk - 1) / chunk;
      split = 1;
      while (split < 8 && split < chunks && row_waves * tiles * split < 4096) split *= 2;
      waves = std::max(4, split);
      row_blocks = (int)((row_waves + waves / split - 1) / (waves / split));
    }
    padded_units = (units + chunk - 1) / chunk * chunk;
    if (!query_tiles) {
      const size_t laid_out = (size_t)padded_units * kUnit * std::min(num_queries, kTile) * planes * 2 + (size_t)groups * kTile * 4 + kTile + 32;
      own = num_queries <= 2 && laid_out <= 32768;
      lds = (own ? (laid_out + 15) / 16 * 16 : 0) + (size_t)(split > 1 ? (split - 1) * (waves / split) : 0) * kRowTiles * 64 * sizeof(float4_t);
    }
  }
};

struct ScoresScratch {
  _Float16* planes;
  signed char* exponents;
  float* sums;
  size_t plane, bytes;
  ScoresScratch(void* memory, int num_queries, const ScoresPlan& p) {
    WorkspaceParts s(memory);
    const size_t queries = p.own ? 0 : (size_t)(num_queries + kTile - 1) / kTile * kTile;
    plane = queries * p.padded_units * kUnit;
    planes = s.part<_Float16>(plane * p.planes);
    exponents = s.part<signed char>(queries);
    sums = s.part<float>(queries * p.groups);
    bytes = s.used();
  }
};

template <typename T, int UC, int GU, int PLANES, bool OWN>
void launch_few(const ScoresArgs& a, const ScoresPlan& p, hipStream_t stream) {
  const long long grid = (long long)a.row_blocks * a.query_blocks;
  want(grid * 64 * p.waves <= 0xffffffffll, "scores: too many rows and queries");
  if (a.offsets) hipLaunchKernelGGL((scores_few_kernel<T, UC, GU, PLANES, false, OWN>), dim3((unsigned)grid), dim3(64 * p.waves), p.lds, stream, a);
  else hipLaunchKernelGGL((scores_few_kernel<T, UC, GU, PLANES, true, OWN>), dim3((unsigned)grid), dim3(64 * p.waves), p.lds, stream, a);
}
template <int UC, int GU>
void launch_few_of(const ScoresArgs& a, const ScoresPlan& p, int query_type, hipStream_t stream) {
  if (p.own && query_type == TYPE_F32) launch_few<float, UC, GU, 2, true>(a, p, stream);
  else if (p.own && query_type == TYPE_F16) launch_few<_Float16, UC, GU, 1, true>(a, p, stream);
  else if (p.own) launch_few<bf16, UC, GU, 1, true>(a, p, stream);
  else if (p.planes == 2) launch_few<float, UC, GU, 2, false>(a, p, stream);
  else launch_few<float, UC, GU, 1, false>(a, p, stream);
}

template <int UC, int GU, int MT, int PLANES>
void launch_many(const ScoresArgs& a, hipStream_t stream) {
  const long long grid = ((long long)a.row_blocks + 7) / 8 * 8 * ((a.query_blocks + a.blocks_each - 1) / a.blocks_each);
  want(grid * 64 * kManyWaves <= 0xffffffffll, "scores: too many rows and queries");
  if (a.offsets) hipLaunchKernelGGL((scores_many_kernel<UC, GU, MT, PLANES, false>), dim3((unsigned)grid), dim3(64 * kManyWaves), 0, stream, a);
  else hipLaunchKernelGGL((scores_many_kernel<UC, GU, MT, PLANES, true>), dim3((unsigned)grid), dim3(64 * kManyWaves), 0, stream, a);
}
template <int UC, int GU, int MT>
void launch_many_of(const ScoresArgs& a, const ScoresPlan& p, hipStream_t stream) {
  if (p.planes == 2) launch_many<UC, GU, MT, 2>(a, stream);
  else launch_many<UC, GU, MT, 1>(a, stream);
}

template <int UC, int GU>
void launch_scores(const ScoresArgs& a, const ScoresPlan& p, int query_type, hipStream_t stream) {
  if constexpr (UC == 2 || UC == 4) {
    if (p.query_tiles == 4) return launch_many_of<UC, GU, 4>(a, p, stream);
    if (p.query_tiles == 3) return launch_many_of<UC, GU, 3>(a, p, stream);
    if (p.query_tiles > 0) return launch_many_of<UC, GU, 2>(a, p, stream);
  }
  launch_few_of<UC, GU>(a, p, query_type, stream);
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

long long cuhnsw_packed_scores_workspace(long long num_rows, int num_dims, int group, int query_type, int num_queries) {
  if (num_rows <= 0 || num_dims <= 0 || group <= 0 || !known_type(query_type) || num_queries <= 0) return 0;
  return (long long)ScoresScratch(nullptr, num_queries, ScoresPlan(num_rows, num_dims, group, query_type, num_queries)).bytes;
}

int cuhnsw_packed_scores_plan(long long num_rows, int num_dims, int group, int query_type, int num_queries, int* out) {
  if (num_rows <= 0 || num_dims <= 0 || group <= 0 || !known_type(query_type) || num_queries <= 0 || !out) return -1;
  const ScoresPlan p(num_rows, num_dims, group, query_type, num_queries);
  out[0] = p.query_tiles;
  out[1] = p.blocks_each;
  out[2] = p.split;
  out[3] = p.own;
  return 0;
}

int cuhnsw_packed_scores(const void* codes, const void* scales, const void* offsets, int scale_type, long long num_rows, int num_dims,
                         int group, const void* queries, int query_type, long long query_stride, int num_queries, float alpha,
                         const float* bias, void* out, int out_type, long long out_stride, void* workspace, long long workspace_bytes,
                         void* stream) {
  return call_guarded([&] {
    check_packed(num_rows, num_dims, group, scale_type);
    want(known_type(query_type) && known_type(out_type), "scores: unknown element type");
    want(out_type == query_type || out_type == TYPE_F32, "scores: the result has the queries' type or is float32");
    want(num_queries >= 0 && query_stride >= 0 && out_stride >= num_rows, "scores: bad sizes");
    if (num_rows == 0 || num_queries == 0) return;
    want(codes && scales && queries && out, "scores: null argument");
    want((reinterpret_cast<uintptr_t>(codes) & 15) == 0, "scores: codes have to be aligned to 16 bytes");
    want(num_rows <= 0x7fffff00ll, "scores: too many rows");
    want(num_queries <= 0xfffff0, "scores: too many queries");  // (a launch has fewer than 2^32 threads)
    ScoresArgs a{};
    a.codes = static_cast<const unsigned char*>(codes);
    a.scales = static_cast<const uint16_t*>(scales);
    a.offsets = static_cast<const uint16_t*>(offsets);
    a.scale_bf16 = scale_type == TYPE_BF16;
    a.num_rows = (int)num_rows;
    a.num_dims = num_dims;
    a.group = group;
    a.units = units_of(num_dims);
    a.groups = (num_dims + group - 1) / group;
    a.queries = queries;
    a.query_stride = query_stride;
    a.num_queries = num_queries;
    a.alpha = alpha;
    a.bias = bias;
    a.out = out;
    a.out_type = out_type;
    a.out_stride = out_stride;
    const ScoresPlan p(num_rows, num_dims, group, query_type, num_queries);
    a.padded_units = p.padded_units;
    a.query_blocks = p.query_blocks;
    a.row_blocks = p.row_blocks;
    a.split = p.split;
    a.blocks_each = p.blocks_each;
    const ScoresScratch w(workspace, num_queries, p);
    want(w.bytes == 0 || (workspace && workspace_bytes >= (long long)w.bytes), "scores: the workspace is too small");
    a.planes = w.planes;
    a.plane = w.plane;
    a.exponents = w.exponents;
    a.sums = w.sums;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (!p.own)
      with_type(query_type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        hipLaunchKernelGGL(prepare_kernel<T>, dim3((unsigned)((num_queries + kTile - 1) / kTile * kTile)), dim3(256), 0, s, a, p.planes);
      });
    const int gu = group / kUnit;
    if (p.chunk == 1) launch_scores<1, 1>(a, p, query_type, s);
    else if (p.chunk == 2) gu == 1 ? launch_scores<2, 1>(a, p, query_type, s) : launch_scores<2, 2>(a, p, query_type, s);
    else if (p.chunk == 3) gu == 1 ? launch_scores<3, 1>(a, p, query_type, s) : gu == 2 ? launch_scores<3, 2>(a, p, query_type, s) : launch_scores<3, 4>(a, p, query_type, s);
    else gu == 1 ? launch_scores<4, 1>(a, p, query_type, s) : gu == 2 ? launch_scores<4, 2>(a, p, query_type, s) : launch_scores<4, 4>(a, p, query_type, s);
    HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
