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
// On the matrix cores, in float16: a code less 8 (or the code) is exact there, and so is a query as one or two planes of
// float16, once a power of two has brought its largest element to [2^14, 2^15): a float32 is the sum of its rounding to 11 bits
// and the rounding of the rest (off by 2^-23 of it, or by 2^-39 of the largest element where that is more), a bfloat16 or a
// float16 is one plane.  Products are summed in 32 bits per group of elements; the group's scale is applied to that sum, so
// no weight is ever rounded.  Offsets meet the group's sum of query elements.
//
// Queries are laid out once per call (prepare_kernel) as the lanes want them: for a tile of up to 16 queries and a unit of 32 elements,
// 16 bytes for every quarter of a unit and query, in the order in which the codes of a word come apart.
constexpr int kTile = 16, kUnit = 32, kRowTiles = 4;  // queries or rows of a matrix product, elements of it; row tiles of a wavefront

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
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
  _Float16* planes;        // [planes][query tile][unit][quarter][query][8]
  size_t plane;            // elements of one plane
  int* exponents;          // [num_queries]: what the scores are to be scaled by
  float* sums;             // [query tile][group][16]: sums of the groups' elements
  int query_blocks, row_blocks, split;
};

template <typename T>
__global__ void __launch_bounds__(256) prepare_kernel(ScoresArgs a, int planes) {
  __shared__ float largest[4];
  const int m = blockIdx.x, tid = threadIdx.x;
  const T* q = static_cast<const T*>(a.queries) + m * a.query_stride;
  int exponent = 14;
  if (!std::is_same_v<T, _Float16>) {
    float most = 0.f;
    for (int k = tid; k < a.num_dims; k += 256) most = fmaxf(most, fabsf(widen(q[k])));
    for (int step = 32; step > 0; step >>= 1) most = fmaxf(most, __shfl_xor(most, step));
    if ((tid & 63) == 0) largest[tid >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(largest[0], largest[1]), fmaxf(largest[2], largest[3]));
    if (most > 0.f && most < INFINITY) exponent = ilogbf(most);
  }
  if (tid == 0) a.exponents[m] = exponent;
  const int tile = m / kTile, i = m % kTile, in_tile = min(kTile, a.num_queries - tile * kTile);
  _Float16* to = a.planes + (size_t)tile * kTile * a.padded_units * kUnit;
  for (int w = tid; w < a.padded_units * 4; w += 256) {  // eight elements: a quarter of a unit
    half8_t high, low;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = w * 8 + (e & 1) * 4 + (e >> 1);  // (0 4 1 5 2 6 3 7)
      const float x = k < a.num_dims ? ldexpf(widen(q[k]), 14 - exponent) : 0.f;
      high[e] = (_Float16)x;
      low[e] = (_Float16)(x - (float)high[e]);
    }
    *reinterpret_cast<half8_t*>(to + ((size_t)w * in_tile + i) * 8) = high;
    if (planes == 2) *reinterpret_cast<half8_t*>(to + a.plane + ((size_t)w * in_tile + i) * 8) = low;
  }
  if (a.offsets)
    for (int g = tid; g < a.groups; g += 256) {
      float sum = 0.f;
      for (int k = g * a.group; k < min(a.num_dims, (g + 1) * a.group); ++k) sum += ldexpf(widen(q[k]), -exponent);
      a.sums[((size_t)tile * a.groups + g) * kTile + i] = sum;
    }
}

// The eight codes of a word, less 8 or as they are, as float16, in the order 0 4 1 5 2 6 3 7: a code behind the exponent of 1024
// is 1024 more (16 times the code behind it for every other one), and what is too much goes off exactly.
template <bool CENTRED>
__device__ inline half8_t codes_of(uint32_t word) {
  constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u, k1024 = 0x64006400u;
  const half2_t low = CENTRED ? half2_t{-1032.f16, -1032.f16} : half2_t{-1024.f16, -1024.f16};
  const half2_t high = CENTRED ? half2_t{-72.f16, -72.f16} : half2_t{-64.f16, -64.f16}, sixteenth = {0.0625f16, 0.0625f16};
  const uint32_t next = word >> 8;
  const half2_t a = __builtin_bit_cast(half2_t, (word & kLow) | k1024) + low;
  const half2_t b = __builtin_elementwise_fma(__builtin_bit_cast(half2_t, (word & kHigh) | k1024), sixteenth, high);
  const half2_t c = __builtin_bit_cast(half2_t, (next & kLow) | k1024) + low;
  const half2_t d = __builtin_elementwise_fma(__builtin_bit_cast(half2_t, (next & kHigh) | k1024), sixteenth, high);
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A wavefront has 64 rows (four tiles of 16) and MT tiles of queries, and goes over the elements in chunks of UC units; `split`
// wavefronts of the workgroup share the chunks of the same rows.  A load of 16 bytes brings a unit's codes to a lane: four such
// slots, one for each quarter of the wavefront, are different units of one row tile, or on short rows of several.  Four lane
// exchanges then give every quarter its quarter of each slot, so one matrix product covers one unit, inside one group.
template <int UC, int GU, int MT, int PLANES, bool CENTRED>
__global__ void __launch_bounds__(512) scores_kernel(ScoresArgs a) {
  constexpr int kGroups = (UC + GU - 1) / GU;  // of a chunk
  constexpr int kAcc = kRowTiles * MT;
  extern __shared__ float4_t partial[];  // [split - 1][row block][kAcc][64]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int j = lane & 15, c = lane >> 4;
  // the query blocks of the same rows one after the other on the same chiplet, whose L2 then holds the rows
  const int turn = blockIdx.x >> 3, per_block = waves / a.split;
  const int block = (turn / a.query_blocks) * 8 + (blockIdx.x & 7), tile0 = (turn % a.query_blocks) * MT;
  const int share = wave % a.split, in_block = wave / a.split;
  const long long row0 = ((long long)block * per_block + in_block) * (kRowTiles * kTile);
  const bool there = row0 < a.num_rows;
  float4_t acc[kRowTiles][MT];
#pragma unroll
  for (int t = 0; t < kRowTiles; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[t][m] = float4_t{0.f, 0.f, 0.f, 0.f};
  if (there) {
    const size_t row_bytes = (size_t)a.units * 16;
    const unsigned char* from[UC];
    int unit_of[UC];
#pragma unroll
    for (int i = 0; i < UC; ++i) {
      const int slot = 4 * i + c;
      const long long row = min(row0 + slot / UC * kTile + j, (long long)a.num_rows - 1);
      unit_of[i] = slot % UC;
      from[i] = a.codes + row * row_bytes;
    }
    long long groups_of[kRowTiles];
#pragma unroll
    for (int t = 0; t < kRowTiles; ++t) groups_of[t] = min(row0 + t * kTile + j, (long long)a.num_rows - 1) * a.groups;
    const _Float16* query_of[MT];
    int in_tile[MT];
    const float* sum_of[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int tile = min(tile0 + m, (a.num_queries - 1) / kTile);
      in_tile[m] = min(kTile, a.num_queries - tile * kTile);
      query_of[m] = a.planes + (size_t)tile * kTile * a.padded_units * kUnit + (c * in_tile[m] + min(j, in_tile[m] - 1)) * 8;
      sum_of[m] = a.sums + (size_t)tile * a.groups * kTile + c * 4;
    }
    const int chunks = (a.units + UC - 1) / UC, per_share = (chunks + a.split - 1) / a.split;
    const int chunk0 = share * per_share, chunk1 = min(chunks, chunk0 + per_share);
    uint4 next[UC];
    auto load = [&](int chunk) {
#pragma unroll
      for (int i = 0; i < UC; ++i)
        next[i] = *reinterpret_cast<const uint4*>(from[i] + min(chunk * UC + unit_of[i], a.units - 1) * 16);
    };
    if (chunk0 < chunk1) load(chunk0);
    for (int chunk = chunk0; chunk < chunk1; ++chunk) {
      uint4 now[UC];
#pragma unroll
      for (int i = 0; i < UC; ++i) now[i] = next[i];
      float scale[kRowTiles][kGroups], offset[kRowTiles][kGroups];
#pragma unroll
      for (int t = 0; t < kRowTiles; ++t)
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const int at = min(chunk * UC / GU + g, a.groups - 1);
          scale[t][g] = half_bits(a.scales[groups_of[t] + at], a.scale_bf16) * 0x1p-14f;
          if (!CENTRED) offset[t][g] = half_bits(a.offsets[groups_of[t] + at], a.scale_bf16);
        }
      half8_t query[UC][MT][PLANES];
#pragma unroll
      for (int u = 0; u < UC; ++u)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int p = 0; p < PLANES; ++p)
            query[u][m][p] = *reinterpret_cast<const half8_t*>(query_of[m] + p * a.plane + (size_t)(chunk * UC + u) * 32 * in_tile[m]);
      if (chunk + 1 < chunk1) load(chunk + 1);
      float4_t temp[MT];
#pragma unroll
      for (int i = 0; i < UC; ++i) {
        const auto ac = __builtin_amdgcn_permlane32_swap(now[i].x, now[i].z, false, false);
        const auto bd = __builtin_amdgcn_permlane32_swap(now[i].y, now[i].w, false, false);
        const auto lo = __builtin_amdgcn_permlane16_swap(ac[0], bd[0], false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap(ac[1], bd[1], false, false);
        const uint32_t slots[4] = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int slot = 4 * i + q, t = slot / UC, u = slot % UC;
          const half8_t codes = codes_of<CENTRED>(slots[q]);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if (u % GU == 0) temp[m] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = PLANES - 1; p >= 0; --p)
              temp[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(query[u][m][p], codes, temp[m], 0, 0, 0);
            if (u % GU == GU - 1 || u == UC - 1) {
              const float s = scale[t][u / GU];
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[t][m][r] = fmaf(s, temp[m][r], acc[t][m][r]);
              if (!CENTRED && chunk * UC / GU + u / GU < a.groups) {
                const float4_t x = *reinterpret_cast<const float4_t*>(sum_of[m] + (chunk * UC / GU + u / GU) * kTile);
                const float o = offset[t][u / GU];
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[t][m][r] = fmaf(o, x[r], acc[t][m][r]);
              }
            }
          }
        }
      }
    }
  }
  if (a.split > 1) {
    if (share > 0)
#pragma unroll
      for (int t = 0; t < kAcc; ++t) partial[(((share - 1) * per_block + in_block) * kAcc + t) * 64 + lane] = acc[t / MT][t % MT];
    __syncthreads();
    if (share > 0) return;
    for (int s = 0; s < a.split - 1; ++s)
#pragma unroll
      for (int t = 0; t < kAcc; ++t) acc[t / MT][t % MT] += partial[((s * per_block + in_block) * kAcc + t) * 64 + lane];
  }
  if (!there) return;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int query = (tile0 + m) * kTile + c * 4 + r;
      if (query >= a.num_queries) continue;
      const int exponent = a.exponents[query];
#pragma unroll
      for (int t = 0; t < kRowTiles; ++t) {
        const long long row = row0 + t * kTile + j;
        if (row >= a.num_rows) continue;
        float y = a.alpha * ldexpf(acc[t][m][r], exponent);
        if (a.bias) y += a.bias[row];
        const long long at = query * a.out_stride + row;
        if (a.out_type == TYPE_F32) static_cast<float*>(a.out)[at] = y;
        else if (a.out_type == TYPE_F16) static_cast<_Float16*>(a.out)[at] = (_Float16)y;
        else static_cast<bf16*>(a.out)[at] = narrow<bf16>(y);
      }
    }
  }
}

struct ScoresScratch {
  _Float16* planes;
  int* exponents;
  float* sums;
  size_t plane, bytes;
  ScoresScratch(void* memory, int num_queries, int padded_units, int planes_wanted, int groups) {
    WorkspaceParts s(memory);
    plane = (size_t)num_queries * padded_units * kUnit;
    planes = s.part<_Float16>(plane * planes_wanted);
    exponents = s.part<int>((size_t)num_queries);
    sums = s.part<float>((size_t)(num_queries + kTile - 1) / kTile * kTile * groups);
    bytes = s.used();
  }
};
inline int units_of(int num_dims) { return (num_dims + kUnit - 1) / kUnit; }
inline int chunk_of(int units) { return std::min(units, 4); }
inline int padded_units_of(int units) { return (units + chunk_of(units) - 1) / chunk_of(units) * chunk_of(units); }
inline int planes_of(int query_type) { return query_type == TYPE_F32 ? 2 : 1; }

template <int UC, int GU, int MT, int PLANES>
void launch_scores(const ScoresArgs& a, int waves, hipStream_t stream) {
  const dim3 grid((unsigned)(((long long)a.row_blocks + 7) / 8 * 8 * a.query_blocks));
  const size_t lds = a.split > 1 ? (size_t)(a.split - 1) * (waves / a.split) * kRowTiles * MT * 64 * sizeof(float4_t) : 0;
  if (a.offsets) hipLaunchKernelGGL((scores_kernel<UC, GU, MT, PLANES, false>), grid, dim3(64 * waves), lds, stream, a);
  else hipLaunchKernelGGL((scores_kernel<UC, GU, MT, PLANES, true>), grid, dim3(64 * waves), lds, stream, a);
}

template <int UC, int GU>
void plan_scores(ScoresArgs& a, int planes, hipStream_t stream) {
  const int tiles = (a.num_queries + kTile - 1) / kTile, mt = tiles == 1 ? 1 : tiles == 2 ? 2 : 4;
  const long long blocks = ((long long)a.num_rows + kRowTiles * kTile - 1) / (kRowTiles * kTile);
  const int chunks = (a.units + UC - 1) / UC;
  a.query_blocks = (tiles + mt - 1) / mt;
  a.split = 1;
  while (mt < 4 && a.split < 8 && a.split < chunks && blocks * a.query_blocks * a.split < 4096) a.split *= 2;
  const int waves = std::max(4, a.split);
  a.row_blocks = (int)((blocks + waves / a.split - 1) / (waves / a.split));
  auto with_planes = [&](auto mts) {
    constexpr int MT = decltype(mts)::value;
    if (planes == 2) launch_scores<UC, GU, MT, 2>(a, waves, stream);
    else launch_scores<UC, GU, MT, 1>(a, waves, stream);
  };
  if (mt == 1) with_planes(std::integral_constant<int, 1>());
  else if (mt == 2) with_planes(std::integral_constant<int, 2>());
  else with_planes(std::integral_constant<int, 4>());
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
  return (long long)ScoresScratch(nullptr, num_queries, padded_units_of(units_of(num_dims)), planes_of(query_type), (num_dims + group - 1) / group).bytes;
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
    a.padded_units = padded_units_of(a.units);
    const int planes = planes_of(query_type);
    const ScoresScratch w(workspace, num_queries, a.padded_units, planes, a.groups);
    want(workspace && workspace_bytes >= (long long)w.bytes, "scores: the workspace is too small");
    a.planes = w.planes;
    a.plane = w.plane;
    a.exponents = w.exponents;
    a.sums = w.sums;
    hipStream_t s = static_cast<hipStream_t>(stream);
    with_type(query_type, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      hipLaunchKernelGGL(prepare_kernel<T>, dim3((unsigned)num_queries), dim3(256), 0, s, a, planes);
    });
    const int uc = chunk_of(a.units), gu = group / kUnit;
    if (uc == 1) plan_scores<1, 1>(a, planes, s);
    else if (uc == 2) gu == 1 ? plan_scores<2, 1>(a, planes, s) : plan_scores<2, 2>(a, planes, s);
    else if (uc == 3) gu == 1 ? plan_scores<3, 1>(a, planes, s) : gu == 2 ? plan_scores<3, 2>(a, planes, s) : plan_scores<3, 4>(a, planes, s);
    else gu == 1 ? plan_scores<4, 1>(a, planes, s) : gu == 2 ? plan_scores<4, 2>(a, planes, s) : plan_scores<4, 4>(a, planes, s);
    HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
