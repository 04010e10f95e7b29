// The 8-bit product on the tensor cores (tcgen05 kind::i8, 32-bit integer sums
// in TMEM).
//
// A cluster of two CTAs computes tiles of 256 channels x up to 256 tokens
// (cta_group::2, M = 256 channels, N = the piece's tokens rounded up to 64):
// CTA r of the pair loads channels ch0 + 128 r .. + 127 of the weight and its
// half of the tokens, the leader issues the MMAs, and each CTA's TMEM receives
// its own 128 channels x all tokens.  The channels are the M side because the
// rows of a group end anywhere: a short piece then costs a smaller N, where
// tokens on the M side would always pay for 256.  The integer sums are exact,
// so one accumulator runs over the whole K; the two 256-column TMEM buffers let
// the epilogue of one tile overlap the next tile's products.
//
// The grid is persistent (one cluster per SM pair); each cluster walks the
// tiles in steps of the cluster count, in groups of eight row pieces so that
// weights and tokens meet in L2.  Where there are fewer tiles than clusters, K
// is cut into `splits` ranges whose 32-bit sums go to a workspace and are added
// and scaled by a second kernel (integers: the order does not matter).
//
// Warp roles per CTA (320 threads): warp 0 TMA producer, warp 1 TMEM owner and
// (leader) MMA issuer, warps 2-9 epilogue.  Every wait is bounded as in the
// Gram kernels; on expiry G2Q_ERR_TIMEOUT goes to the status word and the CTAs
// wind down.
//
// Measured: 16384 x 14336 x 4096 in 596-615 us (3.2 POP/s, tensor pipe 88.4 %
// active; 730-770 us once the card is at its power limit), bound by the pipe;
// 65536 rows of 768 through 128 experts of 2048 channels in 123-129 us, bound by
// the epilogue (6.2k cycles per tile, of which the MMAs need 3.05k); 24 tokens
// through 14336 x 4096 in 17 us with the quantization, bound by reading the weight.
#include "int8.cuh"
#include "rows.cuh"
#include "tc_ptx.cuh"

namespace g2q {
namespace i8 {

using namespace g2q::tc;
using rows::of_f;

constexpr int CH = 256;              // channels per tile (128 per CTA)
constexpr int TOK = 256;             // most tokens per tile, and columns per TMEM buffer
constexpr int KB = 128;              // bytes of K per operand chunk (one swizzled row)
constexpr int KC = 2;                // chunks per pipeline stage
constexpr int OP_BYTES = 128 * KB;   // one operand's chunk in one CTA
constexpr int STAGE_BYTES = KC * 2 * OP_BYTES;
constexpr int STAGES = 3;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int PARTS = EPI_WARPS / 4;        // warps per quadrant, taking turns at blocks of 32 tokens
constexpr int WARP_TOK = TOK / PARTS;       // tokens per warp and tile
constexpr int STRIP_BYTES = 16 * 32 * 2;  // 16 tokens x 32 channels of 2 bytes
constexpr int RASTER = 8;            // row pieces walked together (4 and 16 measured the same)
constexpr int BAR_BYTES = 256;       // barriers, TMEM address, abort flag
static_assert((2 * STAGES + 5) * 8 + 8 <= BAR_BYTES, "barrier area");

// Tensor maps: the weight as [group][chunk][channel][128 bytes] and the tokens as
// [chunk][row][128 bytes] in boxes of KC chunks, the tokens' 32, 64, 96 and 128
// rows high (what a CTA's half of a piece can need; a box is one load and lies
// in shared memory as the MMAs read it).  Where K ends inside a chunk the chunk
// dimension would run into the next row: then K is the innermost dimension and
// the boxes are single chunks.
struct Maps {
  CUtensorMap w, t[4];
};

struct TcArgs {
  Product p;
  int tok;                       // tokens per tile: 64, 128 or 256
  int ch_tiles, nk;              // channel tiles; chunks of K
  int splits, per_split;         // K ranges and chunks in each
  int wide;                      // K is whole chunks: one load per operand and stage
  float per_band;                // 1 / (RASTER * ch_tiles)
  int32_t* part;                 // [splits][M][N] when splits > 1
  long long wait_cycles;
};

// What one cluster works on
struct Tile {
  int row0, rows, group, ch0;
  int k0, k1, split;  // K range in chunks
};

// In shared memory: the first piece and the first row of each group (and what
// would follow the last), so that every role finds its tile by a binary search.
struct Table {
  int32_t* first;  // [groups + 2]
  int32_t* lo;     // [groups + 2]
};

__device__ __forceinline__ void build_table(const Product& p, int tok, const Table& t) {
  const int lane = threadIdx.x & 31;
  const int ends = (int)p.groups + 2;
  long long top = 0;
  for (int g0 = 0; g0 < ends; g0 += 32) {
    const long long lo = group_start(p, g0 + lane, &top);
    if (g0 + lane < ends) t.lo[g0 + lane] = (int)lo;
  }
  __syncwarp();
  int before = 0;
  for (int g0 = 0; g0 < ends; g0 += 32) {
    const int g = g0 + lane;
    const int mine = g + 1 < ends ? (t.lo[g + 1] - t.lo[g] + tok - 1) / tok : 0;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (g < ends) t.first[g] = before + sum - mine;
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
}

// By a whole warp (every lane gets the tile): the way to the next tile is on the
// producer's and the MMA issuer's critical path, so the group is found with two
// ballots and the divisions are few.
__device__ __forceinline__ Tile decode(const TcArgs& a, const Table& t, int w) {
  const int lane = threadIdx.x & 31;
  Tile r;
  r.split = 0;
  if (a.splits > 1) {
    r.split = w % a.splits;
    w /= a.splits;
  }
  const int groups = (int)a.p.groups, pieces = t.first[groups + 1];
  const int band = RASTER * a.ch_tiles;
  int b = (int)((float)w * a.per_band);  // w / band, off by one at most
  b -= b * band > w;
  b += (b + 1) * band <= w;
  const int r0 = b * RASTER, rem = w - b * band;
  const int gsz = pieces - r0;
  int ch, piece;
  if (gsz >= RASTER) {
    ch = rem / RASTER;
    piece = r0 + rem % RASTER;
  } else {
    ch = rem / gsz;
    piece = r0 + (rem - ch * gsz);
  }
  r.ch0 = ch * CH;
  // the last group with first <= piece: first among every 32nd, then in its stretch
  int g = 0;
  if (groups > 1) {
    const unsigned coarse =
        __ballot_sync(0xffffffffu, 32 * lane <= groups && t.first[32 * lane] <= piece);
    g = 32 * (31 - __clz(coarse));
    const unsigned fine =
        __ballot_sync(0xffffffffu, g + lane <= groups && t.first[g + lane] <= piece);
    g += 31 - __clz(fine);
    if (groups == 1024 && t.first[1024] <= piece) g = 1024;
  } else if (t.first[1] <= piece) {
    g = 1;
  }
  r.group = g;
  r.row0 = t.lo[g] + (piece - t.first[g]) * a.tok;
  const int left = t.lo[g + 1] - r.row0;
  r.rows = left < a.tok ? left : a.tok;
  r.k0 = r.split * a.per_split;
  r.k1 = r.k0 + a.per_split < a.nk ? r.k0 + a.per_split : a.nk;
  return r;
}

__device__ __forceinline__ int mma_n(int rows) { return (rows + 63) / 64 * 64; }

// Shared-memory descriptor of a K-major operand: rows of 128 swizzled bytes,
// groups of eight rows 1 KB apart.
__device__ __forceinline__ uint64_t desc_k_sw128(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// kind::i8 instruction descriptor: signed x signed -> s32, both K-major, M = 256
__device__ __forceinline__ uint32_t idesc_i8_m256(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(CH >> 4) << 24);
}

__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t a, uint64_t b,
                                             uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, int x, int y,
                                                 int z, uint32_t mbar_cluster) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(mbar_cluster)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d_pair(uint32_t dst, const CUtensorMap* map, int x, int y,
                                                 int z, int w, uint32_t mbar_cluster) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(mbar_cluster)
      : "memory");
}

// 32 columns (tokens) of 16 TMEM lanes (channels) as matrix fragments: lane l
// holds channels l / 4 and l / 4 + 8, of columns 8 j + 2 (l % 4) and the next in
// r[4 j], r[4 j + 1] and r[4 j + 2], r[4 j + 3].  No wait.
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// The loads' registers pass through, so that nothing reads them before the wait.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&a)[16], uint32_t (&b)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]), "+r"(a[6]), "+r"(a[7]),
                 "+r"(a[8]), "+r"(a[9]), "+r"(a[10]), "+r"(a[11]), "+r"(a[12]), "+r"(a[13]), "+r"(a[14]), "+r"(a[15]),
                 "+r"(b[0]), "+r"(b[1]), "+r"(b[2]), "+r"(b[3]), "+r"(b[4]), "+r"(b[5]), "+r"(b[6]), "+r"(b[7]),
                 "+r"(b[8]), "+r"(b[9]), "+r"(b[10]), "+r"(b[11]), "+r"(b[12]), "+r"(b[13]), "+r"(b[14]), "+r"(b[15])
               :
               : "memory");
}

// Four 8 x 8 matrices of 16-bit values, transposed: lane l gives the address of
// row l % 8 of matrix l / 8.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                                  uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr),
               "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

template <typename S>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  S v[2] = {of_f<S>(a), of_f<S>(b)};
  uint32_t w;
  memcpy(&w, v, 4);
  return w;
}

// The channel scales and biases that one lane needs: one channel where lanes are
// channels (the first entry), four in fragment order.
struct Channels {
  float sb[4], bias[4];
};

template <typename S>
__global__ void __launch_bounds__(THREADS, 1)
    tc_kernel(const __grid_constant__ Maps maps, const TcArgs a) {
  const Product& p = a.p;
  const uint32_t rank = cluster_ctarank();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  // bars[0..S): full (leader's used), [S..2S): empty, [2S..2S+2): accumulator full,
  // [2S+2..2S+4): accumulator drained (leader's used), [2S+4]: MMA completion after an abort
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  uint8_t* strips = smem + STAGES * STAGE_BYTES + BAR_BYTES;  // [EPI_WARPS][STRIP_BYTES]
  float* sa_s = reinterpret_cast<float*>(strips + EPI_WARPS * STRIP_BYTES);  // [EPI_WARPS][2][WARP_TOK]
  Table table;
  table.first = reinterpret_cast<int32_t*>(sa_s + EPI_WARPS * 2 * WARP_TOK);
  table.lo = table.first + p.groups + 2;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES);
  const uint32_t accf0 = smem_u32(bars + 2 * STAGES);
  const uint32_t acce0 = smem_u32(bars + 2 * STAGES + 2);
  const uint32_t drain0 = smem_u32(bars + 2 * STAGES + 4);

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_map(&maps.w);
#pragma unroll
      for (int i = 0; i < 4; ++i) tma_prefetch_map(&maps.t[i]);
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(full0 + 8 * s, 1);
        mbar_init(empty0 + 8 * s, 1);
      }
      for (int b = 0; b < 2; ++b) {
        mbar_init(accf0 + 8 * b, 1);
        mbar_init(acce0 + 8 * b, 2 * EPI_WARPS);
      }
      mbar_init(drain0, 1);
      *abort_flag = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_holder)),
                 "r"(2 * TOK)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else if (warp == 2) {
    build_table(p, a.tok, table);
  }
  fence_before();
  __syncthreads();
  cluster_sync();  // barriers of both CTAs initialised, TMEM allocated in both
  fence_after();
  const uint32_t tmem = *tmem_holder;
  const int total = table.first[p.groups + 1] * a.ch_tiles * a.splits;
  const int step = gridDim.x >> 1;

  launch_dependents();  // the finishing kernel, which waits for this one to end
  int issued = 0;  // stages whose loads this CTA's producer issued
  if (warp == 0) {
    const uint32_t full_lead = mapa_shared(full0, 0);
    // loads of chunks k .. of tile t into stage s (lane 0): the weight's, the tokens'
    auto load_w = [&](const Tile& t, int k, int s) {
      const int nc = a.wide || t.k1 - k >= KC ? KC : t.k1 - k, half = mma_n(t.rows) / 2;
      // the leader's full[s] expects the bytes of both CTAs
      if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2 * nc * (OP_BYTES + half * KB));
      const uint32_t st = smem_u32(smem + s * STAGE_BYTES), fb = full_lead + 8 * s;
      const int y = t.ch0 + 128 * (int)rank;
      if (a.wide) {
        tma_load_4d_pair(st, &maps.w, 0, y, k, t.group, fb);
      } else {
        for (int c = 0; c < nc; ++c)
          tma_load_4d_pair(st + c * OP_BYTES, &maps.w, (k + c) * KB, y, 0, t.group, fb);
      }
    };
    auto load_t = [&](const Tile& t, int k, int s) {
      const int nc = t.k1 - k < KC ? t.k1 - k : KC, half = mma_n(t.rows) / 2;
      const int y = t.row0 + (int)rank * half;
      const uint32_t sb = smem_u32(smem + s * STAGE_BYTES) + KC * OP_BYTES, fb = full_lead + 8 * s;
      const CUtensorMap* m = &maps.t[half / 32 - 1];
      if (a.wide) {
        tma_load_3d_pair(sb, m, 0, y, k, fb);
      } else {
        for (int c = 0; c < nc; ++c) tma_load_3d_pair(sb + c * half * KB, m, (k + c) * KB, y, 0, fb);
      }
    };
    bool ok = true, first = true;
    for (int w = blockIdx.x >> 1; ok && w < total; w += step) {
      const Tile t = decode(a, table, w);
      if (t.group == p.groups) continue;
      int k = t.k0;
      if (first) {
        // the weight does not depend on the kernel before this one (the tokens'
        // quantization): its first stages are on their way while that ends
        for (; issued < STAGES && k < t.k1; k += KC, ++issued)
          if (lane == 0) load_w(t, k, issued);
        wait_predecessor();
        for (int s = 0, kk = t.k0; s < issued; ++s, kk += KC)
          if (lane == 0) load_t(t, kk, s);
        first = false;
      }
      for (; k < t.k1; k += KC) {
        const int s = issued % STAGES;
        const uint32_t ph = (issued / STAGES) & 1;
        ok = mbar_wait(empty0 + 8 * s, ph ^ 1, abort_flag, p.status, a.wait_cycles);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ++issued;
        if (lane == 0) {
          load_w(t, k, s);
          load_t(t, k, s);
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      int it = 0, tc = 0;
      bool ok = true;
      for (int w = blockIdx.x >> 1; ok && w < total; w += step) {
        const Tile t = decode(a, table, w);
        if (t.group == p.groups) continue;
        const int buf = tc & 1;
        const uint32_t use_ph = (uint32_t)((tc >> 1) & 1);
        ++tc;
        ok = mbar_wait(acce0 + 8 * buf, use_ph ^ 1, abort_flag, p.status, a.wait_cycles);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after();
        const uint32_t acc = tmem + (uint32_t)(buf * TOK);
        const int n = mma_n(t.rows);
        const uint32_t idesc = idesc_i8_m256(n);
        for (int k = t.k0; k < t.k1; k += KC) {
          const int s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          ok = mbar_wait(full0 + 8 * s, ph, abort_flag, p.status, a.wait_cycles);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          ++it;
          fence_after();
          if (lane == 0) {
            const int nc = t.k1 - k < KC ? t.k1 - k : KC;
            const uint32_t st = smem_u32(smem + s * STAGE_BYTES);
            for (int c = 0; c < nc; ++c) {
              const uint64_t da = desc_k_sw128(st + c * OP_BYTES);
              const uint64_t db = desc_k_sw128(st + KC * OP_BYTES + c * (n / 2) * KB);
#pragma unroll
              for (int kk = 0; kk < KB / 32; ++kk)  // 32 bytes of K per MMA
                umma_i8_pair(acc, da + 2 * kk, db + 2 * kk, idesc,
                             k > t.k0 || c > 0 || kk > 0 ? 1u : 0u);
            }
            umma_commit_pair(empty0 + 8 * s);
          }
          __syncwarp();
        }
        if (ok && lane == 0) umma_commit_pair(accf0 + 8 * buf);
        __syncwarp();
      }
    }
  } else {
    // warp w reads TMEM lanes 32 (w % 4) .. + 31 (channels) of this CTA; the
    // warps of a quadrant take turns at blocks of 32 tokens
    const int q = warp & 3, part = (warp - 2) / 4;
    const uint32_t acce_lead = mapa_shared(acce0, 0);
    S* out = static_cast<S*>(p.out);
    // 16-bit outputs leave as 16-byte pieces of token rows, through a strip of 16
    // tokens x 32 channels whose pieces are swizzled (piece ^ token / 2) so that
    // neither the transposing stores nor the row reads conflict: the MMAs read
    // their operands from the same shared memory at most of its rate, and 2-byte
    // stores to it took 168 us where this took 142 us (65536 rows of 768 through
    // 128 experts of 2048 channels).  32-bit values leave straight from the
    // registers, a warp's 32 channels being 128 bytes of a token's row.
    const bool frag = sizeof(S) == 2 && a.splits == 1 &&
                      (reinterpret_cast<uintptr_t>(out) & 15) == 0 && p.ldo % 8 == 0 &&
                      p.N % 8 == 0;
    uint8_t* strip = strips + (warp - 2) * STRIP_BYTES;
    const uint32_t st_row = smem_u32(strip) + (lane % 8) * 64 + (((lane / 8) ^ (lane % 8 / 2)) * 16);
    const uint8_t* ld_row = strip + (lane / 4) * 64 + (((lane % 4) ^ (lane / 4 / 2 % 4)) * 16);
    Tile t, next;
    float* sa_w = sa_s + (warp - 2) * 2 * WARP_TOK;
    float sa_next[WARP_TOK / 32];  // lane: one token of each block
    Channels ch_next;
    // a tile's scales are loaded one tile ahead; zeros where there is no such
    // row or channel, and for rows behind the last group
    auto fetch = [&](int w) {
      next = decode(a, table, w);
      const bool zero = next.group == p.groups;
#pragma unroll
      for (int b = 0; b < WARP_TOK / 32; ++b) {
        const int c = 32 * (part + b * PARTS) + lane;
        sa_next[b] = !zero && c < next.rows ? p.sa[next.row0 + c] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (u > 0 && !frag) break;
        const int n = next.ch0 + 128 * (int)rank + q * 32 + (frag ? lane / 4 + 8 * u : lane);
        ch_next.sb[u] = !zero && n < p.N ? p.sb[(long long)next.group * p.N + n] : 0.f;
        ch_next.bias[u] = p.bias && n < p.N ? p.bias[n] : 0.f;
      }
    };
    int tc = 0, turn = 0, w = blockIdx.x >> 1;
    bool ok = true;
    wait_predecessor();  // the tokens' scales
    if (w < total) fetch(w);
    for (; w < total; w += step, ++turn) {
      t = next;
      const Channels ch = ch_next;
      float* sa = sa_w + (turn & 1) * WARP_TOK;
#pragma unroll
      for (int b = 0; b < WARP_TOK / 32; ++b) sa[32 * b + lane] = sa_next[b];
      __syncwarp();
      if (w + step < total) fetch(w + step);
      const bool zero = t.group == p.groups;
      const int buf = tc & 1;
      if (!zero) {
        const uint32_t use_ph = (uint32_t)((tc >> 1) & 1);
        ++tc;
        if (ok) ok = mbar_wait(accf0 + 8 * buf, use_ph, abort_flag, p.status, a.wait_cycles);
        ok = __all_sync(0xffffffffu, ok);
        fence_after();
      }
      const uint32_t base = tmem + (uint32_t)(buf * TOK) + ((uint32_t)(q * 32) << 16);
      const long long n0 = t.ch0 + 128 * (long long)rank + q * 32;
      const long long n = p.N - n0;  // channels of the strip (may be none)
      for (int c0 = 32 * part, cw = 0; c0 < t.rows; c0 += 32 * PARTS, cw += 32) {
        const long long row = t.row0 + c0;
        const int rows = t.rows - c0;
        if (frag) {
          uint32_t r[2][16];
          if (zero) {
#pragma unroll
            for (int u = 0; u < 16; ++u) r[0][u] = r[1][u] = 0;
          } else {
            tmem_ld_16x256b_x4(base + (uint32_t)c0, r[0]);
            tmem_ld_16x256b_x4(base + (uint32_t)c0 + (16u << 16), r[1]);
            tmem_wait_ld(r[0], r[1]);
          }
          if (!ok) continue;
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // 16 tokens
            if (16 * h >= rows) break;
#pragma unroll
            for (int j = 0; j < 2; ++j) {  // 8 of them
              const float2 s2 =
                  *reinterpret_cast<const float2*>(sa + cw + 16 * h + 8 * j + 2 * (lane % 4));
              uint32_t m[4];
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const uint32_t* v = &r[u / 2][8 * h + 4 * j + 2 * (u % 2)];
                m[u] = pack2<S>(scaled((int)v[0], s2.x, ch.sb[u], ch.bias[u]),
                                scaled((int)v[1], s2.y, ch.sb[u], ch.bias[u]));
              }
              stmatrix_x4_trans(st_row + 8 * j * 64, m[0], m[1], m[2], m[3]);
            }
            __syncwarp();
            S* dst = out + (row + 16 * h + lane / 4) * p.ldo + n0 + 8 * (lane % 4);
            const bool in = 8 * (lane % 4) < n;
#pragma unroll
            for (int i = 0; i < 2; ++i)  // 8 tokens
              if (in && 16 * h + 8 * i + lane / 4 < rows)
                *reinterpret_cast<uint4*>(dst + (long long)i * 8 * p.ldo) =
                    *reinterpret_cast<const uint4*>(ld_row + i * 8 * 64);
            __syncwarp();
          }
        } else {
          uint32_t r[32];
          if (zero) {
#pragma unroll
            for (int c = 0; c < 32; ++c) r[c] = 0;
          } else {
            tmem_ld32(base + (uint32_t)c0, r);
          }
          if (!ok || lane >= n) continue;
          if (a.splits > 1) {
            int32_t* dst = a.part + ((long long)t.split * p.M + row) * p.N + n0 + lane;
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (c < rows) dst[c * p.N] = (int)r[c];
          } else {
            S* dst = out + row * p.ldo + n0 + lane;
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (c < rows)
                dst[c * p.ldo] = of_f<S>(scaled((int)r[c], sa[cw + c], ch.sb[0], ch.bias[0]));
          }
        }
      }
      if (!zero) {
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(acce_lead + 8 * buf);
      }
    }
  }
  fence_before();
  __syncthreads();
  if (*abort_flag) {
    // a wait gave up: the leader lets the loads into the stages it armed land and
    // its MMAs finish; the peer, whose loads complete no barrier of its own,
    // allows them a fixed settling time
    if (warp == 0 && lane == 0) {
      if (rank == 0) {
        for (int i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
          mbar_drain(full0 + 8 * (i % STAGES), (i / STAGES) & 1);
      } else if (issued > 0) {
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
      }
    } else if (warp == 1 && lane == 0 && rank == 0) {
      umma_commit_pair(drain0);
      mbar_drain(drain0, 0);
    }
    __syncthreads();
  }
  // neither CTA leaves while the other may still touch its shared memory or TMEM
  cluster_sync();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * TOK)
                 : "memory");
  }
}

// Adds the K ranges' sums and scales them.  The sums and the tokens' scales are
// written by kernels that may still run when this grid starts: no read-only loads.
template <typename S>
__global__ void __launch_bounds__(256)
    finish_kernel(S* __restrict__ out, long long ldo, const int32_t* part, int splits,
                  const float* sa, const float* __restrict__ sb, const float* __restrict__ bias,
                  long long M, long long N) {
  wait_predecessor();
  for (long long m = blockIdx.y; m < M; m += gridDim.y) {
    const float s = sa[m];
    for (long long n = blockIdx.x * 256LL + threadIdx.x; n < N; n += gridDim.x * 256LL) {
      int acc = 0;
#pragma unroll 4
      for (int k = 0; k < splits; ++k) acc += part[(k * M + m) * N + n];
      out[m * ldo + n] = of_f<S>(scaled(acc, s, sb[n], bias ? bias[n] : 0.f));
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

static bool byte_map(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims,
                     const cuuint64_t* strides, int box_rows, int box_chunks) {
  auto enc = encode_fn();
  if (!enc) return false;
  const cuuint32_t box[4] = {KB, (cuuint32_t)box_rows, (cuuint32_t)box_chunks, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static long long up16(long long v) { return (v + 15) / 16 * 16; }

bool tc_takes(const Product& p) {
  return rows::aligned(p.a, 16) && rows::aligned(p.b, 16) && (p.M == 1 || p.lda % 16 == 0) &&
         (p.N == 1 || p.ldb % 16 == 0) && (p.groups == 1 || p.b_gs % 16 == 0);
}

constexpr int kClusters = 74;

// Tokens per tile and K ranges.  Estimated SM cycles of one tile's range: per
// 128-byte chunk of K the larger of the MMAs' (2 cycles per token column) and of
// fetching the CTA's operands from L2 (about 48 bytes per cycle), plus the
// start of a tile and its epilogue; a wave is one range per cluster.  Cutting K
// adds the finishing kernel and the sums' way through L2.  Few tokens and a
// short K come out at small tiles, few tiles and a long K at several ranges.
struct Shape {
  int tok, splits, per;
};

static Shape choose(const Product& p) {
  const int nk = cdiv(p.K, KB);
  const long long ch = (p.N + CH - 1) / CH;
  Shape best = {TOK, 1, nk};
  if (p.offsets) {
    // the pieces are only known on the device: tiles that an average group fills
    const long long avg = p.M / p.groups;
    best.tok = avg > 128 ? 256 : (avg > 64 ? 128 : 64);
    return best;
  }
  double least = 1e300;
  for (int tok = 64; tok <= TOK; tok *= 2) {
    const long long tiles = ((p.M + tok - 1) / tok) * ch;
    for (int want = 1; want <= 16; ++want) {
      const int per = (nk + want - 1) / want, s = (nk + per - 1) / per;
      if (s != want || (want > 1 && per < 4)) continue;
      const double fetch = (128.0 + tok / 2) * KB / 48.0, mma = 2.0 * tok;
      const double chunk = fetch > mma ? fetch : mma;
      const double waves = (double)((tiles * s + kClusters - 1) / kClusters);
      double cost = waves * (per * chunk + 600.0 + 4.0 * tok);
      if (s > 1) cost += 4000.0 + (double)p.M * p.N * (s + 1) * 4.0 / (148 * 24.0);
      if (cost < least) {
        least = cost;
        best = {tok, s, per};
      }
    }
  }
  return best;
}

size_t tc_workspace_bytes(const Product& p) {
  if (!tc_takes(p)) return 0;
  const int s = choose(p).splits;
  return s > 1 ? (size_t)s * p.M * p.N * sizeof(int32_t) : 0;
}

template <typename S>
static int launch_tc(const Maps& maps, const TcArgs& a, long long tiles, bool overlap,
                     cudaStream_t st) {
  const int smem = STAGES * STAGE_BYTES + 1024 + BAR_BYTES + EPI_WARPS * STRIP_BYTES +
                   EPI_WARPS * 2 * WARP_TOK * (int)sizeof(float) +
                   (int)(2 * a.p.groups + 4) * (int)sizeof(int32_t);
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return G2Q_ERR_CUDA;
  static int attr_done[64] = {0};
  if (dev >= 64 || !attr_done[dev]) {
    if (cudaFuncSetAttribute(tc_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             227 * 1024) != cudaSuccess)
      return G2Q_ERR_CUDA;
    if (dev < 64) attr_done[dev] = 1;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (unsigned)(tiles < kClusters ? tiles : kClusters), 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = overlap ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, tc_kernel<S>, maps, a);
  g2q::note_launch();
  if (e == cudaSuccess && a.splits > 1) {
    cudaLaunchConfig_t fin = {};
    fin.gridDim = dim3((unsigned)cdiv(a.p.N, 256), (unsigned)(a.p.M < 65535 ? a.p.M : 65535), 1);
    fin.blockDim = dim3(256, 1, 1);
    fin.stream = st;
    fin.attrs = attr + 1;
    fin.numAttrs = 1;
    e = cudaLaunchKernelEx(&fin, finish_kernel<S>, static_cast<S*>(a.p.out), a.p.ldo,
                           static_cast<const int32_t*>(a.part), a.splits, a.p.sa, a.p.sb, a.p.bias,
                           a.p.M, a.p.N);
    g2q::note_launch();
  }
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return G2Q_ERR_CUDA;
  }
  return G2Q_OK;
}

int tc_product(const Product& p, void* workspace, size_t workspace_bytes, bool overlap,
               cudaStream_t st) {
  TcArgs a;
  a.p = p;
  a.ch_tiles = cdiv(p.N, CH);
  a.nk = cdiv(p.K, KB);
  const Shape shape = choose(p);
  a.tok = shape.tok;
  a.splits = shape.splits;
  a.per_split = shape.per;
  a.part = static_cast<int32_t*>(workspace);
  a.wait_cycles = wait_cycles();
  const size_t need = tc_workspace_bytes(p);
  if (need && (!workspace || workspace_bytes < need || !rows::aligned(workspace, 16)))
    return G2Q_ERR_INVALID_ARG;
  a.wide = p.K % KB == 0;
  a.per_band = 1.f / (float)(RASTER * a.ch_tiles);
  const cuuint64_t lda = (cuuint64_t)(p.M == 1 ? up16(p.K) : p.lda);
  const cuuint64_t ldb = (cuuint64_t)(p.N == 1 ? up16(p.K) : p.ldb);
  const cuuint64_t gs = p.groups > 1 ? (cuuint64_t)p.b_gs : (cuuint64_t)p.N * ldb;
  const cuuint64_t inner = (cuuint64_t)(a.wide ? KB : p.K), chunks = (cuuint64_t)(a.wide ? a.nk : 1);
  const cuuint64_t wd[4] = {inner, (cuuint64_t)p.N, chunks, (cuuint64_t)p.groups};
  const cuuint64_t ws[3] = {ldb, KB, gs};
  const cuuint64_t td[3] = {inner, (cuuint64_t)p.M, chunks};
  const cuuint64_t ts[2] = {lda, KB};
  const int box_chunks = a.wide ? KC : 1;
  Maps maps;
  if (!byte_map(&maps.w, p.b, 4, wd, ws, 128, box_chunks)) return G2Q_ERR_CUDA;
  // the heights that occur: one group has whole pieces and a last one
  const int whole = a.tok / 2, last = (int)((p.M % a.tok + 63) / 64 * 32);
  for (int i = 0; i < 4; ++i) {
    const int rows = 32 * (i + 1);
    if (p.offsets ? rows <= whole : ((rows == whole && p.M >= a.tok) || rows == last)) {
      if (!byte_map(&maps.t[i], p.a, 3, td, ts, rows, box_chunks)) return G2Q_ERR_CUDA;
    } else {
      maps.t[i] = maps.w;  // never read
    }
  }
  const long long tiles = range_slots(p, a.tok) * a.ch_tiles * a.splits;
  // (tile numbers also have to be exact in fp32 to within one band)
  if (tiles > 0xffffffLL) return G2Q_ERR_UNSUPPORTED;
  if (p.out_dtype == G2Q_DTYPE_BF16) return launch_tc<__nv_bfloat16>(maps, a, tiles, overlap, st);
  if (p.out_dtype == G2Q_DTYPE_F16) return launch_tc<__half>(maps, a, tiles, overlap, st);
  return launch_tc<float>(maps, a, tiles, overlap, st);
}

}  // namespace i8
}  // namespace g2q
