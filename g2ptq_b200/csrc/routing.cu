// Expert routing: the (token, slot) pairs of a top-k router sorted by expert,
// token rows copied into that order, expert rows brought back weighted, and
// the gradients of both.
//
//   order       stable sort of the pairs i = t * k + j by expert id; pairs whose
//               id is no expert (negative or >= E) come last
//   position    [T, k]: the pair's row r in that order, or -1 - r where the id
//               is no expert
//   offsets     [E + 1]: expert e has rows offsets[e] .. offsets[e + 1] - 1
//   dispatch    rows[r] = x[t] (zero for pairs without an expert)
//   combine     out[t] = sum_j w[t, j] y[position[t, j]], over pairs with an expert
//   gradients   d y[r] = w[t, j] g[t],  d w[t, j] = <g[t], y[r]>; that of
//               dispatch is combine without weights
//
// Replaces the per-expert gather / scatter of the reference's routed expert
// forward (utils/models/mixins.py:233-259).  Everything is a copy or a short
// dot product, so the row kernels are bound by HBM: each row is read once and
// written once, with all slots of a token handled together.  Measured on rows of
// 2048 bf16: dispatch of 65536 tokens x 8 398 us (6.07 TB/s), combine of 16384 x 8
// 98 us (6.2 TB/s), its gradients 186 us (6.1 TB/s); the sort of 524288 pairs 17 us,
// bound by latency.
#include "rows.cuh"

namespace g2q {
namespace {

using rows::of_f;
using rows::to_f;

// ---------------------------------------------------------------------------
// sort by expert: a counting sort, stable because ranks follow the pair order
// ---------------------------------------------------------------------------

constexpr int SORT_WARPS = 32;
constexpr int SORT_THREADS = 32 * SORT_WARPS;
constexpr int WARP_ITEMS = 128;                      // consecutive pairs per warp
constexpr int CHUNK = SORT_WARPS * WARP_ITEMS;       // pairs per block and round
constexpr long long kMaxExperts = 1024;
constexpr int kMaxSortBlocks = 148;

struct SortArgs {
  const void* ids;
  int wide;  // int64 ids (else int32)
  long long n;
  int E;
  int per;  // pairs per block, a multiple of CHUNK
  int32_t* hist;  // [blocks][E + 1], unused with one block
  int32_t *order, *position, *offsets;
};

__device__ __forceinline__ int key_of(const SortArgs& a, long long i) {
  const long long id = a.wide ? static_cast<const int64_t*>(a.ids)[i]
                              : (long long)static_cast<const int32_t*>(a.ids)[i];
  return id >= 0 && id < a.E ? (int)id : a.E;
}

__global__ void __launch_bounds__(SORT_THREADS) route_count_kernel(SortArgs a) {
  extern __shared__ int32_t cnt[];
  for (int e = threadIdx.x; e <= a.E; e += SORT_THREADS) cnt[e] = 0;
  __syncthreads();
  const long long first = (long long)blockIdx.x * a.per;
  const long long last = first + a.per < a.n ? first + a.per : a.n;
  for (long long i = first + threadIdx.x; i < last; i += SORT_THREADS)
    atomicAdd(&cnt[key_of(a, i)], 1);
  __syncthreads();
  int32_t* h = a.hist + (long long)blockIdx.x * (a.E + 1);
  for (int e = threadIdx.x; e <= a.E; e += SORT_THREADS) h[e] = cnt[e];
}

// The count of the first kernel is what makes a block's ranks independent of
// the other blocks; with one block (at most CHUNK pairs) its own counts do.
template <bool ONE>
__global__ void __launch_bounds__(SORT_THREADS) route_place_kernel(SortArgs a) {
  extern __shared__ int32_t sm[];
  const int E1 = a.E + 1;
  int32_t* base = sm;           // next row of each expert
  int32_t* total = sm + E1;     // pairs of each expert, over all blocks
  uint16_t* part = reinterpret_cast<uint16_t*>(sm + 2 * E1);  // [SORT_WARPS][E1]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned below = (1u << lane) - 1u;

  for (int e = threadIdx.x; e < E1; e += SORT_THREADS) base[e] = total[e] = 0;
  __syncthreads();
  if (!ONE) {
    // threads over experts (adjacent ones adjacent) and, where experts are few,
    // over slices of the blocks
    const int width = E1 < SORT_THREADS ? E1 : SORT_THREADS;
    const int slices = SORT_THREADS / width, s = threadIdx.x / width;
    if (s < slices) {
      for (int e = threadIdx.x % width; e < E1; e += width) {
        int before = 0, all = 0;
#pragma unroll 4
        for (int b = s; b < (int)gridDim.x; b += slices) {
          const int c = a.hist[(long long)b * E1 + e];
          all += c;
          if (b < (int)blockIdx.x) before += c;
        }
        atomicAdd(&base[e], before);
        atomicAdd(&total[e], all);
      }
    }
    __syncthreads();
  }
  auto starts = [&]() {  // base[e] += pairs of the experts before e (one warp)
    int run = 0;
    for (int e0 = 0; e0 < E1; e0 += 32) {
      const int e = e0 + lane;
      const int c = e < E1 ? total[e] : 0;
      int sum = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      if (e < E1) {
        const int start = run + sum - c;
        base[e] += start;
        if (blockIdx.x == 0) a.offsets[e] = start;
      }
      run += __shfl_sync(0xffffffffu, sum, 31);
    }
  };
  if (!ONE && warp == 0) starts();

  const long long first = (long long)blockIdx.x * a.per;
  const long long last = first + a.per < a.n ? first + a.per : a.n;
  for (long long c0 = first; c0 < last || (ONE && c0 == 0); c0 += CHUNK) {
    for (int i = threadIdx.x; i < SORT_WARPS * E1; i += SORT_THREADS) part[i] = 0;
    __syncthreads();
    // rank of each pair among its warp's earlier pairs with the same expert
    uint16_t* mine = part + warp * E1;
    int key[WARP_ITEMS / 32], rank[WARP_ITEMS / 32];
#pragma unroll
    for (int r = 0; r < WARP_ITEMS / 32; ++r) {
      const long long i = c0 + warp * WARP_ITEMS + r * 32 + lane;
      key[r] = i < last ? key_of(a, i) : -1;
    }
#pragma unroll
    for (int r = 0; r < WARP_ITEMS / 32; ++r) {
      const unsigned same = __match_any_sync(0xffffffffu, key[r]);
      const int old = key[r] >= 0 ? mine[key[r]] : 0;
      rank[r] = old + __popc(same & below);
      __syncwarp();
      if (key[r] >= 0 && (same & below) == 0) mine[key[r]] = (uint16_t)(old + __popc(same));
      __syncwarp();
    }
    __syncthreads();
    // counts of the warps become the starts of their pairs within the chunk
    for (int e = threadIdx.x; e < E1; e += SORT_THREADS) {
      int run = 0;
#pragma unroll 8
      for (int w = 0; w < SORT_WARPS; ++w) {
        const int c = part[w * E1 + e];
        part[w * E1 + e] = (uint16_t)run;
        run += c;
      }
      total[e] = run;  // of this chunk, from here on
    }
    __syncthreads();
    if (ONE) {
      if (warp == 0) starts();
      __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < WARP_ITEMS / 32; ++r) {
      if (key[r] < 0) continue;
      const int i = (int)(c0 + warp * WARP_ITEMS + r * 32 + lane);
      const int row = base[key[r]] + mine[key[r]] + rank[r];
      a.order[row] = i;
      a.position[i] = key[r] < a.E ? row : -1 - row;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E1; e += SORT_THREADS) base[e] += total[e];
    if (ONE) break;
  }
}

int sort_blocks(long long n) {
  const long long chunks = (n + CHUNK - 1) / CHUNK;
  return (int)(chunks < 1 ? 1 : (chunks < kMaxSortBlocks ? chunks : kMaxSortBlocks));
}

// ---------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------

// W bytes at a time
template <int W>
struct Piece;
template <>
struct Piece<16> { using T = uint4; };
template <>
struct Piece<4> { using T = uint32_t; };
template <>
struct Piece<2> { using T = uint16_t; };
template <>
struct Piece<1> { using T = uint8_t; };

template <typename V>
__device__ __forceinline__ V zero_piece() {
  V v;
  memset(&v, 0, sizeof(V));
  return v;
}

// One warp per segment of 32 * PL pieces of a token's row: read once, written
// to the row of every slot.
template <int W, int PL>
__global__ void __launch_bounds__(256)
    dispatch_kernel(uint8_t* __restrict__ out, long long ldo, const uint8_t* __restrict__ x,
                    long long ldx, const int32_t* __restrict__ position, long long T, int k,
                    long long n, long long pieces, long long segs) {
  using V = typename Piece<W>::T;
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * 8;
  for (long long item = blockIdx.x * 8LL + (threadIdx.x >> 5); item < T * segs; item += warps) {
    const long long t = item / segs;
    const long long p0 = (item - t * segs) * (32 * PL) + lane;
    const V* src = reinterpret_cast<const V*>(x + t * ldx);
    V v[PL];
#pragma unroll
    for (int i = 0; i < PL; ++i)
      if (p0 + 32 * i < pieces) v[i] = src[p0 + 32 * i];
    for (int j = 0; j < k; ++j) {
      const int p = position[t * k + j];
      const long long row = p < 0 ? -1LL - p : p;
      if (row >= n) continue;
      V* dst = reinterpret_cast<V*>(out + row * ldo);
#pragma unroll
      for (int i = 0; i < PL; ++i)
        if (p0 + 32 * i < pieces) dst[p0 + 32 * i] = p < 0 ? zero_piece<V>() : v[i];
    }
  }
}

// The elements of one piece as fp32
template <typename S, int W>
struct Elems {
  static constexpr int N = W / (int)sizeof(S);
  using V = typename Piece<W>::T;
  __device__ __forceinline__ static void load(float (&f)[N], const V& v) {
#pragma unroll
    for (int u = 0; u < N; ++u) f[u] = to_f<S>(reinterpret_cast<const S*>(&v)[u]);
  }
  __device__ __forceinline__ static V store(const float (&f)[N]) {
    V v;
#pragma unroll
    for (int u = 0; u < N; ++u) reinterpret_cast<S*>(&v)[u] = of_f<S>(f[u]);
    return v;
  }
};

__device__ __forceinline__ float weight_at(const void* w, int dtype, long long i) {
  if (!w) return 1.f;
  if (dtype == G2Q_DTYPE_F32) return static_cast<const float*>(w)[i];
  if (dtype == G2Q_DTYPE_BF16) return to_f(static_cast<const __nv_bfloat16*>(w)[i]);
  return to_f(static_cast<const __half*>(w)[i]);
}

constexpr int SLOTS = 8;  // most slots whose rows are in flight together

// Slots j0 .. j0 + KT - 1 of token t, the same in every lane: their rows (-1
// for none) and weights.
template <int KT>
struct Slots {
  int row[KT];
  float w[KT];

  __device__ __forceinline__ void load(const int32_t* __restrict__ position,
                                       const void* __restrict__ weights, int w_dtype, long long t,
                                       int k, int j0, long long n) {
    const int lane = threadIdx.x & 31;
    int r = -1;
    float v = 0.f;
    if (lane < KT && j0 + lane < k) {
      r = position[t * k + j0 + lane];
      if (r >= n) r = -1;
      if (r >= 0) v = weight_at(weights, w_dtype, t * k + j0 + lane);
    }
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      row[j] = __shfl_sync(0xffffffffu, r, j);
      w[j] = __shfl_sync(0xffffffffu, v, j);
    }
  }
};

// One warp per token (few tokens: per segment of its row, blockIdx.y), U pieces
// per lane in flight for each of KT slots, added in slot order in fp32.  MANY:
// more than KT slots, in rounds.
template <typename S, int W, int KT, int U, bool MANY>
__global__ void __launch_bounds__(256)
    combine_kernel(S* __restrict__ out, long long ldo, const S* __restrict__ y, long long ldy,
                   const int32_t* __restrict__ position, const void* __restrict__ w, int w_dtype,
                   long long T, int k, long long n, int pieces) {
  using L = Elems<S, W>;
  using V = typename L::V;
  const int lane = threadIdx.x & 31;
  for (long long t = blockIdx.x * 8LL + (threadIdx.x >> 5); t < T; t += gridDim.x * 8LL) {
    Slots<KT> s;
    if (!MANY) s.load(position, w, w_dtype, t, k, 0, n);
    for (int p0 = blockIdx.y * (32 * U); p0 < pieces; p0 += gridDim.y * (32 * U)) {
      float acc[U][L::N];
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int u = 0; u < L::N; ++u) acc[i][u] = 0.f;
      for (int j0 = 0; j0 < (MANY ? k : 1); j0 += KT) {
        if (MANY) s.load(position, w, w_dtype, t, k, j0, n);
        V v[KT][U];
#pragma unroll
        for (int j = 0; j < KT; ++j)
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const int p = p0 + 32 * i + lane;
            if (p < pieces && s.row[j] >= 0)
              v[j][i] = reinterpret_cast<const V*>(y + s.row[j] * ldy)[p];
          }
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          if (s.row[j] < 0) continue;
#pragma unroll
          for (int i = 0; i < U; ++i) {
            float f[L::N];
            L::load(f, v[j][i]);
#pragma unroll
            for (int u = 0; u < L::N; ++u) acc[i][u] = fmaf(s.w[j], f[u], acc[i][u]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int p = p0 + 32 * i + lane;
        if (p < pieces) reinterpret_cast<V*>(out + t * ldo)[p] = L::store(acc[i]);
      }
    }
  }
}

// WARPS warps per token: the token's output gradient is read once per round of
// KT slots, every slot's row once for its dot product, and its gradient written.
// Loads in flight are what counts: with eight slots, registers for six CTAs per SM
// instead of four took 184 us for 204 us (16384 x 8 rows of 2048 bf16).
template <typename S, int W, int KT, int U, int WARPS>
__global__ void __launch_bounds__(128, KT == 8 ? (U == 1 ? 6 : 3) : 4)
    combine_bwd_kernel(S* __restrict__ gy, long long ldgy, void* __restrict__ gw,
                       const S* __restrict__ g, long long ldg, const S* __restrict__ y,
                       long long ldy, const int32_t* __restrict__ position,
                       const void* __restrict__ w, int w_dtype, long long T, int k, long long n,
                       int pieces) {
  using L = Elems<S, W>;
  using V = typename L::V;
  constexpr int TOKENS = 4 / WARPS;  // per block
  __shared__ float part[4][KT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = warp % WARPS;
  for (long long t0 = (long long)blockIdx.x * TOKENS; t0 < T; t0 += (long long)gridDim.x * TOKENS) {
    const long long t = t0 + warp / WARPS;
    if (WARPS == 1 && t >= T) break;
    const V* gr = reinterpret_cast<const V*>(g + t * ldg);
    for (int j0 = 0; j0 < k; j0 += KT) {
      Slots<KT> s;
      s.load(position, w, w_dtype, t, k, j0, n);
      // rows of pairs without an expert, whose gradient is zero
      int bare[KT];
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        bare[j] = -1;
        if (s.row[j] < 0 && j0 + j < k && gy) {
          const int p = position[t * k + j0 + j];
          if (p < 0 && -1LL - p < n) bare[j] = -1 - p;
        }
      }
      float dot[KT];
#pragma unroll
      for (int j = 0; j < KT; ++j) dot[j] = 0.f;
      for (int p0 = sub * (32 * U); p0 < pieces; p0 += WARPS * (32 * U)) {
        V gv[U], v[KT][U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int p = p0 + 32 * i + lane;
          gv[i] = zero_piece<V>();
          if (p < pieces) gv[i] = gr[p];
        }
        if (gw) {
#pragma unroll
          for (int j = 0; j < KT; ++j)
#pragma unroll
            for (int i = 0; i < U; ++i) {
              const int p = p0 + 32 * i + lane;
              v[j][i] = zero_piece<V>();
              if (p < pieces && s.row[j] >= 0)
                v[j][i] = reinterpret_cast<const V*>(y + s.row[j] * ldy)[p];
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int p = p0 + 32 * i + lane;
          float gf[L::N];
          L::load(gf, gv[i]);
#pragma unroll
          for (int j = 0; j < KT; ++j) {
            if (gw) {
              float f[L::N];
              L::load(f, v[j][i]);
#pragma unroll
              for (int u = 0; u < L::N; ++u)
                if (p < pieces && s.row[j] >= 0) dot[j] = fmaf(gf[u], f[u], dot[j]);
            }
            if (gy && p < pieces) {
              if (s.row[j] >= 0) {
                float f[L::N];
#pragma unroll
                for (int u = 0; u < L::N; ++u) f[u] = s.w[j] * gf[u];
                reinterpret_cast<V*>(gy + s.row[j] * ldgy)[p] = L::store(f);
              } else if (bare[j] >= 0) {
                reinterpret_cast<V*>(gy + bare[j] * ldgy)[p] = zero_piece<V>();
              }
            }
          }
        }
      }
      if (gw) {
        float mine = 0.f;  // lane j: slot j0 + j's dot product
#pragma unroll
        for (int j = 0; j < KT; ++j) {
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
          if (lane == j) mine = dot[j];
        }
        if (WARPS > 1) {
          if (lane < KT) part[warp][lane] = mine;
          __syncthreads();
          mine = 0.f;
          if (lane < KT) {
#pragma unroll
            for (int q = 0; q < WARPS; ++q) mine += part[warp - sub + q][lane];
          }
          __syncthreads();
        }
        if (sub == 0 && lane < KT && j0 + lane < k) {
          const long long i = t * k + j0 + lane;
          if (w_dtype == G2Q_DTYPE_F32) static_cast<float*>(gw)[i] = mine;
          else if (w_dtype == G2Q_DTYPE_BF16)
            static_cast<__nv_bfloat16*>(gw)[i] = of_f<__nv_bfloat16>(mine);
          else static_cast<__half*>(gw)[i] = of_f<__half>(mine);
        }
      }
    }
  }
}

// The widest piece that every row of the buffers can be cut into.
int piece_bytes(long long row_bytes, int eb, const void* a, long long lda, const void* b,
                long long ldb, const void* c, long long ldc) {
  const long long all = row_bytes | (lda * eb) | (ldb * eb) | (ldc * eb) |
                        (long long)(reinterpret_cast<uintptr_t>(a) |
                                    reinterpret_cast<uintptr_t>(b) |
                                    reinterpret_cast<uintptr_t>(c));
  return all % 16 == 0 ? 16 : (all % 4 == 0 ? 4 : (all % 2 == 0 ? 2 : 1));
}

unsigned warp_grid(long long items) {
  long long blocks = (items + 7) / 8;
  if (blocks > 148 * 64) blocks = 148 * 64;
  return (unsigned)(blocks < 1 ? 1 : blocks);
}

template <int W>
int launch_dispatch(void* out, long long ldo, const void* x, long long ldx, const int32_t* position,
                    long long T, int k, long long row_bytes, cudaStream_t st) {
  const long long pieces = row_bytes / W;
  uint8_t* o = static_cast<uint8_t*>(out);
  const uint8_t* s = static_cast<const uint8_t*>(x);
  // four pieces per lane where the rows are many enough to fill the machine
  if (T * ((pieces + 127) / 128) >= 148 * 16) {
    const long long segs = (pieces + 127) / 128;
    dispatch_kernel<W, 4><<<warp_grid(T * segs), 256, 0, st>>>(o, ldo, s, ldx, position, T, k,
                                                               T * k, pieces, segs);
  } else {
    const long long segs = (pieces + 31) / 32;
    dispatch_kernel<W, 1><<<warp_grid(T * segs), 256, 0, st>>>(o, ldo, s, ldx, position, T, k,
                                                               T * k, pieces, segs);
  }
  G2Q_CHECK_LAUNCH();
  return G2Q_OK;
}

template <typename S, int W, int KT, int U, bool MANY>
int launch_combine_k(void* out, long long ldo, const void* y, long long ldy,
                     const int32_t* position, const void* w, int w_dtype, long long T, int k,
                     int pieces, cudaStream_t st) {
  // a row is cut into segments only where whole rows would leave warp slots idle
  const long long most = (pieces + 32 * U - 1) / (32 * U);
  long long segs = (148 * 32 + T - 1) / T;
  if (segs > most) segs = most;
  long long gx = (T + 7) / 8;
  if (gx > 148 * 64) gx = 148 * 64;
  combine_kernel<S, W, KT, U, MANY><<<dim3((unsigned)gx, (unsigned)segs), 256, 0, st>>>(
      static_cast<S*>(out), ldo, static_cast<const S*>(y), ldy, position, w, w_dtype, T, k, T * k,
      pieces);
  G2Q_CHECK_LAUNCH();
  return G2Q_OK;
}

template <typename S, int W>
int launch_combine(void* out, long long ldo, const void* y, long long ldy, const int32_t* position,
                   const void* w, int w_dtype, long long T, int k, long long C, cudaStream_t st) {
  const long long all = C * (long long)sizeof(S) / W;
  if (all > 0x7fffff00LL) return G2Q_ERR_UNSUPPORTED;
  const int pieces = (int)all;
  // pieces in flight per slot: eight loads of 16 bytes per lane, more of the
  // narrower ones (rows of odd sizes)
  constexpr int X = W == 16 ? 1 : 4;
#define G2Q_COMBINE(KT, U, MANY) \
  launch_combine_k<S, W, KT, U, MANY>(out, ldo, y, ldy, position, w, w_dtype, T, k, pieces, st)
  if (k == 1) return G2Q_COMBINE(1, 4 * (X / 2 + X % 2), false);
  if (k == 2) return G2Q_COMBINE(2, 4 * (X / 2 + X % 2), false);
  if (k <= 4) return G2Q_COMBINE(4, 2 * X, false);
  if (k <= SLOTS) return G2Q_COMBINE(8, X, false);
  return G2Q_COMBINE(8, X, true);
#undef G2Q_COMBINE
}

template <typename S, int W, int KT, int U>
int launch_combine_bwd_k(void* gy, long long ldgy, void* gw, const void* g, long long ldg,
                         const void* y, long long ldy, const int32_t* position, const void* w,
                         int w_dtype, long long T, int k, int pieces, cudaStream_t st) {
  // one warp per token where the rows are short or the tokens fill the machine
  if (pieces <= 32 * U || T >= 148 * 16) {
    long long blocks = (T + 3) / 4;
    if (blocks > 148 * 64) blocks = 148 * 64;
    combine_bwd_kernel<S, W, KT, U, 1><<<(unsigned)blocks, 128, 0, st>>>(
        static_cast<S*>(gy), ldgy, gw, static_cast<const S*>(g), ldg, static_cast<const S*>(y), ldy,
        position, w, w_dtype, T, k, T * k, pieces);
  } else {
    combine_bwd_kernel<S, W, KT, U, 4><<<(unsigned)T, 128, 0, st>>>(
        static_cast<S*>(gy), ldgy, gw, static_cast<const S*>(g), ldg, static_cast<const S*>(y), ldy,
        position, w, w_dtype, T, k, T * k, pieces);
  }
  G2Q_CHECK_LAUNCH();
  return G2Q_OK;
}

template <typename S, int W>
int launch_combine_bwd(void* gy, long long ldgy, void* gw, const void* g, long long ldg,
                       const void* y, long long ldy, const int32_t* position, const void* w,
                       int w_dtype, long long T, int k, long long C, cudaStream_t st) {
  const long long all = C * (long long)sizeof(S) / W;
  if (all > 0x7fffff00LL) return G2Q_ERR_UNSUPPORTED;
  const int pieces = (int)all;
  constexpr int X = W == 16 ? 1 : 4;
#define G2Q_BWD(KT, U) \
  launch_combine_bwd_k<S, W, KT, U>(gy, ldgy, gw, g, ldg, y, ldy, position, w, w_dtype, T, k, \
                                    pieces, st)
  if (k == 1) return G2Q_BWD(1, 4 * (X / 2 + X % 2));
  if (k == 2) return G2Q_BWD(2, 4 * (X / 2 + X % 2));
  if (k <= 4) return G2Q_BWD(4, 2 * (X / 2 + X % 2));
  return G2Q_BWD(8, X / 2 + X % 2);
#undef G2Q_BWD
}

bool routed_shape_ok(long long T, long long k, long long C) {
  return T >= 0 && k > 0 && C > 0 && k <= 0x7fffffffLL && (T == 0 || k <= 0x7fffffffLL / T);
}

bool weight_dtype_ok(int d) { return rows::elem_bytes(d) != 0; }

}  // namespace
}  // namespace g2q

using namespace g2q;

extern "C" size_t g2q_route_workspace_bytes(int64_t n, int64_t E) {
  if (n <= 0 || E <= 0 || n <= CHUNK) return 0;
  return (size_t)sort_blocks(n) * (size_t)(E + 1) * sizeof(int32_t);
}

extern "C" int g2q_route(int32_t* order, int32_t* position, int32_t* offsets, const void* ids,
                         int ids_wide, int64_t n, int64_t E, void* workspace,
                         size_t workspace_bytes, void* stream) {
  if (n < 0 || E <= 0 || !offsets || (ids_wide != 0 && ids_wide != 1)) return G2Q_ERR_INVALID_ARG;
  if (E > kMaxExperts || n > 0x7fffffffLL - CHUNK) return G2Q_ERR_UNSUPPORTED;
  if (n > 0 && (!order || !position || !ids)) return G2Q_ERR_INVALID_ARG;
  const size_t need = g2q_route_workspace_bytes(n, E);
  if (need && (!workspace || workspace_bytes < need)) return G2Q_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const int blocks = sort_blocks(n);
  SortArgs a = {ids, ids_wide, n, (int)E, 0, static_cast<int32_t*>(workspace), order, position,
                offsets};
  const long long chunks = (n + CHUNK - 1) / CHUNK;
  a.per = (int)((chunks + blocks - 1) / blocks) * CHUNK;
  const int smem = (int)(2 * (E + 1) * sizeof(int32_t) + SORT_WARPS * (E + 1) * sizeof(uint16_t));
  if (n <= CHUNK) {
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(route_place_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             smem) != cudaSuccess)
      return G2Q_ERR_CUDA;
    route_place_kernel<true><<<1, SORT_THREADS, smem, st>>>(a);
    G2Q_CHECK_LAUNCH();
    return G2Q_OK;
  }
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(route_place_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           smem) != cudaSuccess)
    return G2Q_ERR_CUDA;
  route_count_kernel<<<blocks, SORT_THREADS, (E + 1) * sizeof(int32_t), st>>>(a);
  G2Q_CHECK_LAUNCH();
  route_place_kernel<false><<<blocks, SORT_THREADS, smem, st>>>(a);
  G2Q_CHECK_LAUNCH();
  return G2Q_OK;
}

extern "C" int g2q_dispatch_rows(void* out, int64_t ldo, const void* x, int64_t ldx, int elem_size,
                                 const int32_t* position, int64_t T, int64_t k, int64_t C,
                                 void* stream) {
  if (!routed_shape_ok(T, k, C) || ldo < C || ldx < C ||
      (elem_size != 1 && elem_size != 2 && elem_size != 4))
    return G2Q_ERR_INVALID_ARG;
  if (T == 0) return G2Q_OK;
  if (!out || !x || !position) return G2Q_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const long long es = elem_size, rb = C * es;
  switch (piece_bytes(rb, elem_size, out, ldo, x, ldx, x, ldx)) {
    case 16: return launch_dispatch<16>(out, ldo * es, x, ldx * es, position, T, (int)k, rb, st);
    case 4: return launch_dispatch<4>(out, ldo * es, x, ldx * es, position, T, (int)k, rb, st);
    case 2: return launch_dispatch<2>(out, ldo * es, x, ldx * es, position, T, (int)k, rb, st);
    default: return launch_dispatch<1>(out, ldo * es, x, ldx * es, position, T, (int)k, rb, st);
  }
}

#define G2Q_BY_PIECE(FN, S, W, ...)                       \
  switch (W) {                                            \
    case 16: return FN<S, 16>(__VA_ARGS__);               \
    case 4: return FN<S, 4>(__VA_ARGS__);                 \
    default: return FN<S, (int)sizeof(S)>(__VA_ARGS__);   \
  }

extern "C" int g2q_combine_rows(void* out, int64_t ldo, const void* y, int64_t ldy, int dtype,
                                const int32_t* position, const void* weights, int w_dtype,
                                int64_t T, int64_t k, int64_t C, void* stream) {
  const int eb = rows::elem_bytes(dtype);
  if (!eb || !routed_shape_ok(T, k, C) || ldo < C || ldy < C ||
      (weights && !weight_dtype_ok(w_dtype)))
    return G2Q_ERR_INVALID_ARG;
  if (T == 0) return G2Q_OK;
  if (!out || !y || !position) return G2Q_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const int W = piece_bytes(C * eb, eb, out, ldo, y, ldy, y, ldy);
  if (dtype == G2Q_DTYPE_BF16) {
    G2Q_BY_PIECE(launch_combine, __nv_bfloat16, W, out, ldo, y, ldy, position, weights, w_dtype, T,
                 (int)k, C, st)
  } else if (dtype == G2Q_DTYPE_F16) {
    G2Q_BY_PIECE(launch_combine, __half, W, out, ldo, y, ldy, position, weights, w_dtype, T, (int)k,
                 C, st)
  }
  G2Q_BY_PIECE(launch_combine, float, W, out, ldo, y, ldy, position, weights, w_dtype, T, (int)k, C,
               st)
}

extern "C" int g2q_combine_rows_backward(void* grad_y, int64_t ldgy, void* grad_w,
                                         const void* grad, int64_t ldg, const void* y, int64_t ldy,
                                         int dtype, const int32_t* position, const void* weights,
                                         int w_dtype, int64_t T, int64_t k, int64_t C,
                                         void* stream) {
  const int eb = rows::elem_bytes(dtype);
  if (!eb || !routed_shape_ok(T, k, C) || ldg < C || (grad_y && ldgy < C) ||
      (grad_w && ldy < C) || !weight_dtype_ok(w_dtype))
    return G2Q_ERR_INVALID_ARG;
  if (T == 0 || (!grad_y && !grad_w)) return G2Q_OK;
  if (!grad || !position || !weights || (grad_w && !y)) return G2Q_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const int W = piece_bytes(C * eb, eb, grad, ldg, grad_y ? grad_y : grad, grad_y ? ldgy : ldg,
                            grad_w ? y : grad, grad_w ? ldy : ldg);
  if (dtype == G2Q_DTYPE_BF16) {
    G2Q_BY_PIECE(launch_combine_bwd, __nv_bfloat16, W, grad_y, ldgy, grad_w, grad, ldg, y, ldy,
                 position, weights, w_dtype, T, (int)k, C, st)
  } else if (dtype == G2Q_DTYPE_F16) {
    G2Q_BY_PIECE(launch_combine_bwd, __half, W, grad_y, ldgy, grad_w, grad, ldg, y, ldy, position,
                 weights, w_dtype, T, (int)k, C, st)
  }
  G2Q_BY_PIECE(launch_combine_bwd, float, W, grad_y, ldgy, grad_w, grad, ldg, y, ldy, position,
               weights, w_dtype, T, (int)k, C, st)
}
