// The 8-bit product for a handful of tokens: the weight streams through once and
// its bytes are all the work, so what counts is loads in flight and a short way
// from launch to result.  The tensor-core tiles (int8_tc.cu) spend several
// microseconds on TMEM, clusters, the ring and a second kernel for K ranges.
//
// A CTA of eight warps takes 16 * RG channels; the warps of one 16-channel group
// share K in turns of 64 * DEPTH bytes.  A lane loads 16 bytes of channels g and g + 8
// (g = lane / 4) and 16 bytes of token g, and multiplies them with two
// mma.sync.m16n8k32 (int8): the order of K inside a step is free as long as both
// operands use the same, so 16 consecutive bytes serve as the four words that a
// lane owes two steps.  The warps' integer sums meet in shared memory.
//
// Measured: one token through 4096 x 4096 in 4.5 us with the weight in L2 and 6.0 us
// from memory, 14336 x 4096 in 13.8 us (4.3 TB/s), eight tokens through 14336 x
// 16384 in 48 us (4.9 TB/s; a plain sum of as many bytes reads 5.3): bound by
// reading the weight.
//
// A single token's codes are made by the kernel itself (FUSED): every CTA makes
// them in shared memory, behind its first weight loads.
#include "int8.cuh"
#include "int8_quant.cuh"
#include "tc_ptx.cuh"

namespace g2q {
namespace i8 {

using rows::of_f;

constexpr int SW = 8;       // warps per CTA
constexpr int STEP = 64;    // bytes of K per warp and step

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                       uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Bytes k .. k + 15 of a row of K bytes, missing ones zero.  ONCE: read a single
// time (the weight), so not kept (23.5 -> 20.8 us for four tokens' 128 experts).
// Else the tokens' codes: the kernel before this one may write them while this grid
// is already resident, so they are not read-only for its whole life and take an
// ordinary load, behind wait_predecessor().
template <bool ONCE>
__device__ __forceinline__ uint4 load16(const int8_t* row, long long k, long long K) {
  if (k + 16 <= K) {
    const uint4* v = reinterpret_cast<const uint4*>(row + k);
    return ONCE ? __ldcs(v) : *v;
  }
  uint32_t w[4] = {0, 0, 0, 0};
  if (k < K) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (k + i < K) w[i / 4] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i % 4));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The slot-th group that has rows (counting the rows behind the last group as
// one more); false where there are fewer.  By each warp alone.  Groups as
// group_start has them: while the offsets ascend within [0, M] that is what stands
// there; from the first that does not, every warp that needs it takes the way of the
// running maximum.
__device__ __forceinline__ bool find_group(const Product& p, int slot, int* group, long long* lo,
                                           long long* hi) {
  const int lane = threadIdx.x & 31, wanted = slot;
  for (int g0 = 0; g0 <= p.groups; g0 += 128) {
    int from[4], to[4];
    bool ascend = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int g = g0 + 32 * i + lane;
      from[i] = to[i] = 0;
      if (g <= p.groups) {
        from[i] = g == 0 ? 0 : p.offsets[g];
        to[i] = g < p.groups ? p.offsets[g + 1] : (int)p.M;
        ascend = ascend && from[i] <= to[i] && to[i] <= p.M;
      }
    }
    if (!__all_sync(0xffffffffu, ascend)) {
      // pieces of M rows: one to a group
      Range r = {0, -1, 0};
      find_range(p, wanted, (int)p.M, &r);
      const int src = __ffs(__ballot_sync(0xffffffffu, r.rows >= 0)) - 1;
      const long long row0 = __shfl_sync(0xffffffffu, r.row0, src);
      const int rows = __shfl_sync(0xffffffffu, r.rows, src);
      *group = __shfl_sync(0xffffffffu, r.group, src);
      *lo = row0;
      *hi = row0 + rows;
      return rows > 0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned has = __ballot_sync(0xffffffffu, to[i] > from[i]);
      const int count = __popc(has);
      if (slot < count) {
        // the lane with `slot` set lanes before it
        const bool mine = (has >> lane & 1u) && __popc(has & ((1u << lane) - 1u)) == slot;
        const int src = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
        *group = g0 + 32 * i + src;
        *lo = __shfl_sync(0xffffffffu, from[i], src);
        *hi = __shfl_sync(0xffffffffu, to[i], src);
        return true;
      }
      slot -= count;
    }
  }
  return false;
}

struct Input {  // the token before quantization (FUSED)
  const void* x;
  bool vec;
};

// Bytes of one token's codes in shared memory, zeros behind the last column.
__host__ __device__ __forceinline__ int fused_bytes(const Product& p) {
  return (int)((p.K + 127) / 128 * 128);
}

// CTAs per SM: two of the variants with the most loads in flight, else three, four
// where a 16-bit token is quantized (64 registers: 448 CTAs of 14336 channels x 4096
// are one wave, 13.8 us; 72 registers took 16.6).
template <typename X, int RG, int MG, bool FUSED>
constexpr int stream_ctas() {
  return RG == 1 || MG == 2 ? 2 : (FUSED && sizeof(X) == 2 ? 4 : 3);
}

// MG groups of eight tokens at a time; FUSED: one token.
template <typename S, typename X, int RG, int MG, bool FUSED>
__global__ void __launch_bounds__(32 * SW, stream_ctas<X, RG, MG, FUSED>())
    stream_kernel(const Product p, const Input in) {
  constexpr int KS = SW / RG, TOKENS = 8 * MG, CHANNELS = 16 * RG;
  // steps whose loads are in flight together (eight instead of four: 5.3 -> 5.0 us
  // for eight tokens through 4096 x 4096; with more channels per CTA slower)
  constexpr int DEPTH = RG == 1 && MG == 1 ? 8 : 4;
  extern __shared__ uint4 dyn[];  // FUSED: the token's codes
  __shared__ int red[KS][CHANNELS][TOKENS + 1];
  __shared__ float sa_s[TOKENS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rg = warp % RG, ks = warp / RG, g = lane / 4, t4 = lane % 4;
  int group = 0;
  const long long n0 = (long long)blockIdx.x * CHANNELS;
  long long lo = 0, hi = p.M;
  if (p.offsets) {
    // the grid ends after the kernel before it even if no CTA has rows
    if (blockIdx.x == 0 && blockIdx.y == 0) tc::wait_predecessor();
    if (!find_group(p, blockIdx.y, &group, &lo, &hi)) return;
  }
  S* out = static_cast<S*>(p.out);
  if (group == p.groups) {  // rows behind the last group
    for (long long i = threadIdx.x; i < (hi - lo) * CHANNELS; i += 32 * SW) {
      const long long n = n0 + i % CHANNELS;
      if (n < p.N) out[(lo + i / CHANNELS) * p.ldo + n] = of_f<S>(0.f);
    }
    return;
  }
  const int8_t* b = p.b + (long long)group * p.b_gs;
  const long long c0 = n0 + 16 * rg + g;
  // channels that do not exist read the last one's bytes; their sums go nowhere
  const int8_t* w0 = b + (c0 < p.N ? c0 : p.N - 1) * p.ldb;
  const int8_t* w1 = b + (c0 + 8 < p.N ? c0 + 8 : p.N - 1) * p.ldb;
  // a warp's steps in flight are neighbours in K: 64 * DEPTH bytes of each row
  const int turns = (int)((p.K + STEP * DEPTH - 1) / (STEP * DEPTH));
  uint4 wa[DEPTH], wb[DEPTH];
  auto load_w = [&](int turn) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const long long k = ((long long)turn * DEPTH + d) * STEP + 16 * t4;
      wa[d] = load16<true>(w0, k, p.K);
      wb[d] = load16<true>(w1, k, p.K);
    }
  };
  load_w(ks);
  tc::wait_predecessor();  // the tokens' codes and scales; the weight does not depend on them

  int8_t* codes = reinterpret_cast<int8_t*>(dyn);
  if (FUSED) {
    __shared__ unsigned tops[SW];
    quantize_row<X, 32 * SW>(codes, fused_bytes(p), sa_s, static_cast<const X*>(in.x), (int)p.K,
                             in.vec, tops);
    __syncthreads();
  }

  for (long long m0 = lo; m0 < hi; m0 += TOKENS) {
    const int have = hi - m0 < TOKENS ? (int)(hi - m0) : TOKENS;
    if (!FUSED && threadIdx.x < TOKENS)
      sa_s[threadIdx.x] = threadIdx.x < have ? p.sa[m0 + threadIdx.x] : 0.f;
    int acc[MG][4];
#pragma unroll
    for (int j = 0; j < MG; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0;
    for (int turn = ks; turn < turns; turn += KS) {
      if (turn != ks || m0 != lo) load_w(turn);
      uint4 tok[DEPTH][MG];
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const long long k = ((long long)turn * DEPTH + d) * STEP + 16 * t4;
#pragma unroll
        for (int j = 0; j < MG; ++j) {
          const int m = 8 * j + g;
          tok[d][j] = make_uint4(0, 0, 0, 0);
          if (m < have && k < p.K) {
            if (FUSED) tok[d][j] = *reinterpret_cast<const uint4*>(codes + k);
            else tok[d][j] = load16<false>(p.a + (m0 + m) * p.lda, k, p.K);
          }
        }
      }
#pragma unroll
      for (int d = 0; d < DEPTH; ++d)
#pragma unroll
        for (int j = 0; j < MG; ++j) {
          mma_s8(acc[j], wa[d].x, wb[d].x, wa[d].y, wb[d].y, tok[d][j].x, tok[d][j].y);
          mma_s8(acc[j], wa[d].z, wb[d].z, wa[d].w, wb[d].w, tok[d][j].z, tok[d][j].w);
        }
    }
    // lane: channels g, g + 8; tokens 2 t4, 2 t4 + 1 of each group
#pragma unroll
    for (int j = 0; j < MG; ++j) {
      red[ks][16 * rg + g][8 * j + 2 * t4] = acc[j][0];
      red[ks][16 * rg + g][8 * j + 2 * t4 + 1] = acc[j][1];
      red[ks][16 * rg + g + 8][8 * j + 2 * t4] = acc[j][2];
      red[ks][16 * rg + g + 8][8 * j + 2 * t4 + 1] = acc[j][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < CHANNELS * have; i += 32 * SW) {
      const int c = i % CHANNELS, m = i / CHANNELS;
      const long long n = n0 + c;
      if (n >= p.N) continue;
      int sum = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s) sum += red[s][c][m];
      out[(m0 + m) * p.ldo + n] = of_f<S>(
          scaled(sum, sa_s[m], p.sb[(long long)group * p.N + n], p.bias ? p.bias[n] : 0.f));
    }
    if (m0 + TOKENS < hi) __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Longest row that every CTA quantizes for itself: 4096 columns took 5.0 us with
// and 5.3 us without the separate kernel, 14336 columns 16.9 and 15.5 us; four
// tokens of 4096 columns 8.2 and 5.3 us.
constexpr long long kFusedColumns = 8192;

bool stream_takes(const Product& p) {
  if (!tc_takes(p)) return false;  // the same alignment
  // one group: two groups of eight tokens; groups: few rows each on average, whose
  // weights are then read once as long as the rows are spread evenly (a group of
  // many rows reads its weight again for every eight of them)
  if (p.offsets) return p.M <= 2 * p.groups && p.M <= 4096;
  // more than eight tokens double the work per weight byte: 14336 channels x 4096
  // took 20.6 us here and 17.1 us on the tiles, 4096 x 4096 6.4 and 11.5 us
  return p.M <= (p.N <= 8192 ? 16 : 8);
}

bool stream_quantizes(const Product& p) {
  return stream_takes(p) && !p.offsets && p.M == 1 && p.K <= kFusedColumns;
}

template <typename S, typename X, int RG, int MG, bool FUSED>
static int launch_stream(const Product& p, const Input& in, bool overlap, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cdiv(p.N, 16 * RG), 
                     p.offsets ? (unsigned)(p.groups < p.M ? p.groups + 1 : p.M) : 1, 1);
  cfg.blockDim = dim3(32 * SW, 1, 1);
  cfg.dynamicSmemBytes = FUSED ? fused_bytes(p) : 0;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = overlap ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, stream_kernel<S, X, RG, MG, FUSED>, p, in);
  g2q::note_launch();
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return G2Q_ERR_CUDA;
  }
  return G2Q_OK;
}

template <typename S>
static int stream_out(const Product& p, bool overlap, cudaStream_t st) {
  const Input none = {nullptr, false};
  if (p.offsets) return launch_stream<S, float, 4, 1, false>(p, none, overlap, st);
  // every warp needs a turn of K (512 bytes of it for eight tokens and one channel
  // group per CTA, else 256): 14336 channels x 1024 took 11.1 us with eight warps
  // per group and 5.5 us with four
  if (p.M <= 8) {
    if (p.K >= 4096) return launch_stream<S, float, 1, 1, false>(p, none, overlap, st);
    if (p.K >= 1024) return launch_stream<S, float, 2, 1, false>(p, none, overlap, st);
    return launch_stream<S, float, 4, 1, false>(p, none, overlap, st);
  }
  if (p.K >= 2048) return launch_stream<S, float, 1, 2, false>(p, none, overlap, st);
  return launch_stream<S, float, 4, 2, false>(p, none, overlap, st);
}

int stream_product(const Product& p, bool overlap, cudaStream_t st) {
  if (p.out_dtype == G2Q_DTYPE_BF16) return stream_out<__nv_bfloat16>(p, overlap, st);
  if (p.out_dtype == G2Q_DTYPE_F16) return stream_out<__half>(p, overlap, st);
  return stream_out<float>(p, overlap, st);
}

template <typename S, typename X>
static int stream_in_out(const Product& p, const Input& in, cudaStream_t st) {
  // more CTAs than are resident at once: half as many, which quantize the token
  // half as often (14336 x 4096 13.8 us, with 16 channels per CTA 17.1 us; 4096 x
  // 4096 5.7 and 4.6 us)
  if (p.K < 1024) return launch_stream<S, X, 4, 1, true>(p, in, false, st);
  if (p.K < 4096 || p.N > 148 * 3 * 16) return launch_stream<S, X, 2, 1, true>(p, in, false, st);
  return launch_stream<S, X, 1, 1, true>(p, in, false, st);
}

template <typename X>
static int stream_in(const Product& p, const Input& in, cudaStream_t st) {
  if (p.out_dtype == G2Q_DTYPE_BF16) return stream_in_out<__nv_bfloat16, X>(p, in, st);
  if (p.out_dtype == G2Q_DTYPE_F16) return stream_in_out<__half, X>(p, in, st);
  return stream_in_out<float, X>(p, in, st);
}

int stream_linear(const Product& p, const void* x, int x_dtype, cudaStream_t st) {
  const Input in = {x, rows::aligned(x, 16)};
  if (x_dtype == G2Q_DTYPE_BF16) return stream_in<__nv_bfloat16>(p, in, st);
  if (x_dtype == G2Q_DTYPE_F16) return stream_in<__half>(p, in, st);
  return stream_in<float>(p, in, st);
}

}  // namespace i8
}  // namespace g2q
