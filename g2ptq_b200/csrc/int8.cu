// 8-bit linears: per-token int8 quantization of activations and the product
// of int8 codes with a scale per token and per channel.
//
//   scale_t = max_c |x_tc| / 127            q_tc = round(x_tc / scale_t)
//   y_tn    = scale_t * wscale_n * sum_c q_tc w_nc + bias_n
//
// The sums are exact in 32-bit integers (|q w| <= 128 * 128, C <= 131071); the
// only roundings are the conversion of the sum to fp32, the two scalings, the
// bias and the output type.
#include "int8.cuh"
#include "int8_quant.cuh"
#include "tc_ptx.cuh"

namespace g2q {
namespace i8 {

using rows::of_f;

// ---------------------------------------------------------------------------
// quantization of token rows
// ---------------------------------------------------------------------------

// G threads per row, UNITS units of 16 elements per thread kept in registers
// between the maximum and the codes (one read of x): 16384 x 4096 bf16 in 38 us
// (5.3 TB/s), about even between HBM and issue slots (55 % of each).  What is left of a row --
// the units beyond UNITS * G, a part of a unit at its end -- goes element by
// element and is read a second time.  VEC: rows on 16-byte boundaries.
template <typename S, int G, int UNITS, bool VEC>
__global__ void __launch_bounds__(G > 128 ? G : 128)
    quantize_kernel(int8_t* __restrict__ codes, long long ldq, float* __restrict__ scale_out,
                    const S* __restrict__ x, long long ldx, long long T, int C, bool qvec) {
  constexpr int BLOCK = G > 128 ? G : 128;
  constexpr int PER = BLOCK / G;  // rows per block
  tc::launch_dependents();  // a product that overlaps waits for this kernel to end
  const int tid = threadIdx.x % G;
  const long long t = blockIdx.x * (long long)PER + threadIdx.x / G;
  const bool live = t < T;
  const S* row = x + (live ? t : 0) * ldx;
  int whole = live ? C / 16 : 0;  // units that the unrolled loops take
  whole = whole < UNITS * G ? whole : UNITS * G;
  const int units = live ? (C + 15) / 16 : 0;

  Unit<S> u[UNITS];
#pragma unroll
  for (int k = 0; k < UNITS; ++k)
    if (tid + k * G < whole) {
      if (VEC) u[k].load(row + 16 * (tid + k * G));
      else u[k].load_any(row + 16 * (tid + k * G));
    }
  unsigned top = 0;
#pragma unroll
  for (int k = 0; k < UNITS; ++k)
    if (tid + k * G < whole) top = max_bits<S>(top, u[k].top_bits());
  top = top_of<S>(top);
  for (int i = whole + tid; i < units; i += G) {
    Unit<S> v;
    v.load_part(row + 16LL * i, C - 16 * i);
    top = max(top, top_of<S>(v.top_bits()));
  }
  if constexpr (G < 32) {  // the lanes of this row
    top = __reduce_max_sync(((1u << G) - 1u) << ((threadIdx.x & 31) / G * G), top);
  } else {
    top = __reduce_max_sync(0xffffffffu, top);
  }
  if constexpr (G > 32) {
    __shared__ unsigned warp_top[BLOCK / 32];
    if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
    __syncthreads();
    const int w0 = (threadIdx.x / G) * (G / 32);
#pragma unroll
    for (int w = 0; w < G / 32; ++w) top = max(top, warp_top[w0 + w]);
  }
  if (!live) return;
  RowScale rs;
  const bool finite = row_scale(top, &rs);
  if (tid == 0) scale_out[t] = finite ? rs.scale : __uint_as_float(0x7fc00000u);
  int8_t* qrow = codes + t * ldq;
#pragma unroll
  for (int k = 0; k < UNITS; ++k)
    if (tid + k * G < whole)
      store_codes<S>(qrow + 16 * (tid + k * G), u[k], 16, qvec, rs, finite);
  for (int i = whole + tid; i < units; i += G) {
    Unit<S> v;
    v.load_part(row + 16LL * i, C - 16 * i);
    store_codes<S>(qrow + 16LL * i, v, C - 16 * i, qvec, rs, finite);
  }
}

template <typename S, int G, int UNITS>
static int launch_quantize(int8_t* codes, long long ldq, float* scale, const S* x, long long ldx,
                           long long T, long long C, cudaStream_t st) {
  constexpr int BLOCK = G > 128 ? G : 128;
  const long long blocks = (T + BLOCK / G - 1) / (BLOCK / G);
  if (blocks > 0x7fffffffLL || C > 0x7fffff00LL) return G2Q_ERR_UNSUPPORTED;
  const bool xvec = rows::aligned(x, 16) && (T <= 1 || (ldx * (long long)sizeof(S)) % 16 == 0);
  const bool qvec = rows::aligned(codes, 16) && (T <= 1 || ldq % 16 == 0);
  if (xvec)
    quantize_kernel<S, G, UNITS, true><<<(unsigned)blocks, BLOCK, 0, st>>>(codes, ldq, scale, x,
                                                                           ldx, T, (int)C, qvec);
  else
    quantize_kernel<S, G, UNITS, false><<<(unsigned)blocks, BLOCK, 0, st>>>(codes, ldq, scale, x,
                                                                            ldx, T, (int)C, qvec);
  G2Q_CHECK_LAUNCH();
  return G2Q_OK;
}

template <typename S>
static int quantize_rows(int8_t* codes, long long ldq, float* scale, const void* x, long long ldx,
                         long long T, long long C, cudaStream_t st) {
  const S* xs = static_cast<const S*>(x);
  // Few rows: sixteen warps each, so that more SMs and more loads are at work.
  if (T < 2 * 148) return launch_quantize<S, 512, 2>(codes, ldq, scale, xs, ldx, T, C, st);
  // Else as few lanes per row as its elements in registers allow (128 bytes of them
  // per thread): the row's reduction and division serve the most elements.
  constexpr int U = sizeof(S) == 2 ? 4 : 2;
  if (C <= 256 * U) return launch_quantize<S, 16, U>(codes, ldq, scale, xs, ldx, T, C, st);
  if (C <= 512 * U) return launch_quantize<S, 32, U>(codes, ldq, scale, xs, ldx, T, C, st);
  if (C <= 1024 * U) return launch_quantize<S, 64, U>(codes, ldq, scale, xs, ldx, T, C, st);
  if (C <= 2048 * U) return launch_quantize<S, 128, U>(codes, ldq, scale, xs, ldx, T, C, st);
  if (C <= 4096 * U) return launch_quantize<S, 256, U>(codes, ldq, scale, xs, ldx, T, C, st);
  return launch_quantize<S, 512, U>(codes, ldq, scale, xs, ldx, T, C, st);
}

int quantize_tokens(int8_t* codes, long long ldq, float* scale, const void* x, int dtype,
                    long long ldx, long long T, long long C, cudaStream_t st) {
  if (dtype == G2Q_DTYPE_BF16)
    return quantize_rows<__nv_bfloat16>(codes, ldq, scale, x, ldx, T, C, st);
  if (dtype == G2Q_DTYPE_F16) return quantize_rows<__half>(codes, ldq, scale, x, ldx, T, C, st);
  return quantize_rows<float>(codes, ldq, scale, x, ldx, T, C, st);
}

// ---------------------------------------------------------------------------
// product on the CUDA cores: operands of any alignment (a weight with rows at odd
// strides; 16384 x 14336 x 4096 took 18.8 ms)
// ---------------------------------------------------------------------------

constexpr int ST = 64;   // tile edge (tokens and channels)
constexpr int SKW = 16;  // 32-bit words of K per step

// The word of codes k .. k+3 of a row, missing ones zero.
__device__ __forceinline__ int load_word(const int8_t* row, long long k, long long K, bool vec) {
  if (vec && k + 4 <= K) return *reinterpret_cast<const int*>(row + k);
  int v = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (k + i < K) v |= (static_cast<int>(row[k + i]) & 255) << (8 * i);
  return v;
}

template <typename S>
__global__ void __launch_bounds__(256) simt_kernel(Product p, bool avec, bool bvec) {
  __shared__ int as[ST][SKW + 1], bs[ST][SKW + 1];
  __shared__ Range range;
  if (threadIdx.x < 32) find_range(p, blockIdx.y, ST, &range);
  __syncthreads();
  const Range r = range;
  if (r.rows <= 0) return;
  const long long n0 = (long long)blockIdx.x * ST;
  S* out = static_cast<S*>(p.out);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  int acc[4][4] = {};
  if (r.group < p.groups) {
    const int8_t* b = p.b + r.group * p.b_gs;
    for (long long k0 = 0; k0 < p.K; k0 += 4 * SKW) {
      for (int i = threadIdx.x; i < ST * SKW; i += 256) {
        const int row = i / SKW, w = i % SKW;
        const long long k = k0 + 4 * w;
        as[row][w] = row < r.rows && k < p.K
                         ? load_word(p.a + (r.row0 + row) * p.lda, k, p.K, avec) : 0;
        bs[row][w] = n0 + row < p.N && k < p.K
                         ? load_word(b + (n0 + row) * p.ldb, k, p.K, bvec) : 0;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < SKW; ++w) {
        int av[4], bv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) av[i] = as[ty + 16 * i][w];
#pragma unroll
        for (int j = 0; j < 4; ++j) bv[j] = bs[tx + 16 * j][w];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(av[i], bv[j], acc[i][j]);
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = ty + 16 * i;
    if (row >= r.rows) continue;
    const long long m = r.row0 + row;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long n = n0 + tx + 16 * j;
      if (n >= p.N) continue;
      float v = 0.f;  // rows behind the last group
      if (r.group < p.groups)
        v = scaled(acc[i][j], p.sa[m], p.sb[r.group * p.N + n], p.bias ? p.bias[n] : 0.f);
      out[m * p.ldo + n] = of_f<S>(v);
    }
  }
}

static int simt_product(const Product& p, cudaStream_t st) {
  const long long tiles = range_slots(p, ST);
  const long long cols = (p.N + ST - 1) / ST;
  if (tiles > 65535 || cols > 0x7fffffffLL) return G2Q_ERR_UNSUPPORTED;
  const bool avec = rows::aligned(p.a, 4) && p.lda % 4 == 0;
  const bool bvec = rows::aligned(p.b, 4) && p.ldb % 4 == 0 && p.b_gs % 4 == 0;
  const dim3 grid((unsigned)cols, (unsigned)tiles);
  if (p.out_dtype == G2Q_DTYPE_BF16)
    simt_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p, avec, bvec);
  else if (p.out_dtype == G2Q_DTYPE_F16)
    simt_kernel<__half><<<grid, 256, 0, st>>>(p, avec, bvec);
  else
    simt_kernel<float><<<grid, 256, 0, st>>>(p, avec, bvec);
  G2Q_CHECK_LAUNCH();
  return G2Q_OK;
}

static int product(const Product& p, void* workspace, size_t workspace_bytes, bool overlap,
                   cudaStream_t st) {
  if (stream_takes(p)) return stream_product(p, overlap, st);
  return tc_takes(p) ? tc_product(p, workspace, workspace_bytes, overlap, st) : simt_product(p, st);
}

// Workspace of a product whose operands are aligned.
static size_t product_workspace(const Product& p) {
  return stream_takes(p) ? 0 : tc_workspace_bytes(p);
}

static size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Workspace of a linear whose weight is aligned: the tokens' codes, their scales,
// the product's own.
static size_t linear_workspace(const Product& p) {
  if (stream_quantizes(p)) return 0;
  const size_t M = (size_t)p.M, ld = (size_t)((p.K + 15) / 16 * 16);
  return up256(M * ld) + up256(M * sizeof(float)) + product_workspace(p);
}

static int check(const Product& p) {
  if (!rows::elem_bytes(p.out_dtype) || p.M < 0 || p.N <= 0 || p.K <= 0 || p.groups <= 0)
    return G2Q_ERR_INVALID_ARG;
  if (p.K > kMaxK || p.M > kMaxRows || p.N > kMaxRows || p.groups > kMaxGroups)
    return G2Q_ERR_UNSUPPORTED;
  if (p.M == 0) return G2Q_OK;
  if (!p.out || !p.a || !p.sa || !p.b || !p.sb || p.lda < p.K || p.ldb < p.K || p.ldo < p.N ||
      (p.groups > 1 && (!p.offsets || p.b_gs < p.N * p.ldb)))
    return G2Q_ERR_INVALID_ARG;
  return G2Q_OK;
}

}  // namespace i8
}  // namespace g2q

using namespace g2q;

extern "C" int g2q_quantize_tokens(int8_t* codes, int64_t ldq, float* scale, const void* x,
                                   int dtype, int64_t ldx, int64_t T, int64_t C, void* stream) {
  if (!rows::elem_bytes(dtype) || T < 0 || C <= 0 || ldx < C || ldq < C) return G2Q_ERR_INVALID_ARG;
  if (T == 0) return G2Q_OK;
  if (!codes || !scale || !x) return G2Q_ERR_INVALID_ARG;
  return i8::quantize_tokens(codes, ldq, scale, x, dtype, ldx, T, C, (cudaStream_t)stream);
}

extern "C" size_t g2q_int8_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > i8::kMaxK || M > i8::kMaxRows ||
      N > i8::kMaxRows)
    return 0;
  i8::Product p = {};
  p.lda = p.ldb = (K + 15) / 16 * 16;
  p.groups = 1;
  p.M = M;
  p.N = N;
  p.K = K;
  return i8::product_workspace(p);
}

extern "C" int g2q_int8_matmul(void* out, int out_dtype, int64_t ldo, const int8_t* a, int64_t lda,
                               const float* a_scale, const int8_t* b, int64_t ldb,
                               const float* b_scale, const float* bias, int64_t M, int64_t N,
                               int64_t K, void* workspace, size_t workspace_bytes, int* status,
                               void* stream) {
  i8::Product p = {out, out_dtype, ldo, a, lda, a_scale, b, ldb, 0, b_scale, bias, nullptr, 1,
                   M, N, K, status};
  G2Q_TRY(i8::check(p));
  if (M == 0) return G2Q_OK;
  return i8::product(p, workspace, workspace_bytes, false, (cudaStream_t)stream);
}

extern "C" int g2q_int8_matmul_grouped(void* out, int out_dtype, int64_t ldo, const int8_t* a,
                                       int64_t lda, const float* a_scale, const int8_t* b,
                                       int64_t ldb, int64_t b_gs, const float* b_scale,
                                       const int32_t* offsets, int64_t G, int64_t M, int64_t N,
                                       int64_t K, int* status, void* stream) {
  i8::Product p = {out, out_dtype, ldo, a, lda, a_scale, b, ldb, b_gs, b_scale, nullptr, offsets,
                   G, M, N, K, status};
  if (!offsets) return G2Q_ERR_INVALID_ARG;
  G2Q_TRY(i8::check(p));
  if (M == 0) return G2Q_OK;
  return i8::product(p, nullptr, 0, false, (cudaStream_t)stream);
}

extern "C" size_t g2q_int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t G,
                                                  int aligned) {
  if (M <= 0 || N <= 0 || K <= 0 || G < 0 || K > i8::kMaxK || M > i8::kMaxRows ||
      N > i8::kMaxRows || G > i8::kMaxGroups)
    return 0;
  i8::Product p = {};
  p.lda = p.ldb = (K + 15) / 16 * 16;
  p.b_gs = p.ldb * N;
  p.groups = G > 0 ? G : 1;
  p.offsets = G > 0 ? reinterpret_cast<const int32_t*>(16) : nullptr;  // only whether there are any
  p.M = M;
  p.N = N;
  p.K = K;
  p.b = reinterpret_cast<const int8_t*>(aligned ? 256 : 257);
  size_t need = i8::linear_workspace(p);
  // the tensor-core product ignores the row stride of a single channel and the stride
  // of a single expert: with `aligned` 0 because of such a stride it still runs
  if (!aligned && (N == 1 || G == 1)) {
    p.b = reinterpret_cast<const int8_t*>(256);
    const size_t other = i8::linear_workspace(p);
    need = other > need ? other : need;
  }
  return need;
}

extern "C" int g2q_int8_linear(void* out, int out_dtype, int64_t ldo, const void* x, int x_dtype,
                               int64_t ldx, const int8_t* b, int64_t ldb, int64_t b_gs,
                               const float* b_scale, const float* bias, const int32_t* offsets,
                               int64_t G, int64_t M, int64_t N, int64_t K, void* workspace,
                               size_t workspace_bytes, int* status, void* stream) {
  const int64_t ld = (K + 15) / 16 * 16;
  if (!rows::elem_bytes(x_dtype) || ldx < K || G < 0 || (G > 0) != (offsets != nullptr) ||
      (G > 0 && bias))
    return G2Q_ERR_INVALID_ARG;
  // aligned stand-ins for the operands that the workspace will hold
  i8::Product p = {out, out_dtype, ldo, reinterpret_cast<int8_t*>(256), ld,
                   reinterpret_cast<float*>(256), b, ldb, b_gs, b_scale, bias, offsets,
                   G > 0 ? G : 1, M, N, K, status};
  G2Q_TRY(i8::check(p));
  if (M == 0) return G2Q_OK;
  const size_t need = i8::linear_workspace(p);
  if (!x || (need && (!workspace || !rows::aligned(workspace, 16) || workspace_bytes < need)))
    return G2Q_ERR_INVALID_ARG;
  if (i8::stream_quantizes(p))
    return i8::stream_linear(p, x, x_dtype, (cudaStream_t)stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const size_t code_bytes = i8::up256((size_t)M * (size_t)ld);
  const size_t scale_bytes = i8::up256((size_t)M * sizeof(float));
  float* scale = reinterpret_cast<float*>(ws + code_bytes);
  p.a = reinterpret_cast<int8_t*>(ws);
  p.sa = scale;
  G2Q_TRY(i8::quantize_tokens(reinterpret_cast<int8_t*>(ws), ld, scale, x, x_dtype, ldx, M, K,
                              (cudaStream_t)stream));
  return i8::product(p, ws + code_bytes + scale_bytes, workspace_bytes - code_bytes - scale_bytes,
                     true, (cudaStream_t)stream);
}
