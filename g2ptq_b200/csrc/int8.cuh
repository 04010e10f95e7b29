// The 8-bit product's arguments and the mapping of work to row ranges.
#pragma once

#include "common.cuh"

namespace g2q {
namespace i8 {

constexpr long long kMaxK = 131071;     // 128 * 128 * K fits an int32 sum
constexpr long long kMaxGroups = 1024;  // experts
constexpr long long kMaxRows = 0x7fff0000LL;  // row and channel indexes stay in 32 bits

// out[m, n] = sa[m] * sb[g, n] * sum_k a[m, k] * b[g, n, k] + bias[n], with
// g the group of row m: rows offsets[g] .. offsets[g + 1] - 1 (offsets NULL:
// one group of all rows).  Rows behind the last group give zeros.
struct Product {
  void* out;
  int out_dtype;
  long long ldo;
  const int8_t* a;
  long long lda;
  const float* sa;
  const int8_t* b;
  long long ldb, b_gs;
  const float* sb;
  const float* bias;
  const int32_t* offsets;
  long long groups;
  long long M, N, K;
  int* status;
};

// A piece of at most `tile` rows that share one group; group == groups: rows
// behind the last group; rows <= 0: nothing to do.
struct Range {
  long long row0;
  int rows, group;
};

// Number of pieces that any offsets can give (the grid's extent).
static inline long long range_slots(const Product& p, int tile) {
  const long long full = (p.M + tile - 1) / tile;
  return p.offsets ? full + (p.groups < p.M ? p.groups : p.M) : full;
}

// First row of group g (of group == groups: of the rows behind the last one;
// beyond: M), for 32 neighbouring g of a warp's lanes in ascending calls with
// *top = 0 before the first: the running maximum of the offsets within [0, M],
// so that the groups partition [0, M] whatever the offsets hold.
__device__ __forceinline__ long long group_start(const Product& p, long long g, long long* top) {
  const int lane = threadIdx.x & 31;
  long long v = 0;
  if (g > p.groups || (!p.offsets && g > 0)) v = p.M;
  else if (g > 0) v = p.offsets[g];
  v = v < *top ? *top : (v > p.M ? p.M : v);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o && up > v) v = up;
  }
  *top = __shfl_sync(0xffffffffu, v, 31);
  return v;
}

// The slot-th piece of `tile` rows, counted through the groups in order (one
// warp; one lane writes *out).
__device__ __forceinline__ void find_range(const Product& p, long long slot, int tile, Range* out) {
  const int lane = threadIdx.x & 31;
  long long before = 0, top = 0;
  for (long long g0 = 0; g0 <= p.groups; g0 += 31) {
    // 31 groups and the next one's start
    const long long g = g0 + lane;
    long long from = top;
    const long long lo = group_start(p, g, &from);
    const long long hi = __shfl_down_sync(0xffffffffu, lo, 1);
    const long long mine = lane < 31 && g <= p.groups ? (hi - lo + tile - 1) / tile : 0;
    long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const long long first = before + sum - mine;
    const bool here = slot >= first && slot < first + mine;
    if (here) {
      const long long row0 = lo + (slot - first) * tile, left = hi - row0;
      *out = Range{row0, (int)(left < tile ? left : tile), (int)g};
    }
    if (__any_sync(0xffffffffu, here)) return;
    before += __shfl_sync(0xffffffffu, sum, 31);
    top = __shfl_sync(0xffffffffu, lo, 30);
  }
  if (lane == 0) *out = Range{0, 0, 0};
}

// The sum scaled: converted to fp32 (rounded once), times the token's and the
// channel's scale, plus the bias.
__device__ __forceinline__ float scaled(int acc, float sa, float sb, float bias) {
  return fmaf(__int2float_rn(acc) * sa, sb, bias);
}

// The tensor-core product (int8_tc.cu): whether it takes these operands (bases
// and row strides multiples of 16 bytes), the workspace it needs, the launch
// (`overlap`: it may start while the stream's last kernel, which wrote a and
// sa and nothing else that it reads, is still running).
bool tc_takes(const Product& p);
size_t tc_workspace_bytes(const Product& p);
int tc_product(const Product& p, void* workspace, size_t workspace_bytes, bool overlap,
               cudaStream_t st);

// The product for a handful of tokens (int8_stream.cu): whether it takes these
// operands (aligned like above), the launch, and the same with a single token
// quantized by the kernel itself.
bool stream_takes(const Product& p);
int stream_product(const Product& p, bool overlap, cudaStream_t st);
bool stream_quantizes(const Product& p);
int stream_linear(const Product& p, const void* x, int x_dtype, cudaStream_t st);

}  // namespace i8
}  // namespace g2q
