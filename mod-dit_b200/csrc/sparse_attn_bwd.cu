// Gradients of block-sparse attention for sm_100a.  The probabilities are computed again from the forward's log-sum-exp:
//   P = exp(scale * q.k - lse)   dP = dout v^T   dS = P * (dP - delta),  delta = sum(dout * out) per row
//   dv = P^T dout                dk = scale * dS^T q                     dq = scale * dS k
//
// Two kinds of work item, each of which owns its output rows, so nothing is added through memory and no result depends on
// the order in which blocks run:
//   key item    one tile of 128 keys, walks the query tiles that attend to it: four products per tile
//               S^T = K Q^T, dP^T = V dO^T (both 128 x 128, keys are the tensor-memory lanes), dV += P^T dO, dK += dS^T Q
//   query item  one tile of 128 queries, walks its key tiles: three products per tile
//               S = Q K^T, dP = dO V^T, dQ += dS K
// That is seven products where one pass over the pairs would need five; that pass would add every tile's 64 KB of float32 dQ
// into memory with atomics, in an order that varies (tensor memory would have room for it, with 64 streamed rows at a time).
// Keeping dS for a product of its own would take 32 KB per kept tile (12 GB for three heads of 115,456 tokens).
//
// Both kinds work alike: a block holds two fixed tiles (F0, F1 = K, V or Q, dO) and streams blocks of 64 rows of two tensors
// (X0, X1 = Q, dO or K, V):   S = F0 X0^T,  dP = F1 X1^T,  acc1 += P X1 (key items),  acc0 += dS X0.
// P and dS stay in tensor memory, 16 bits wide, over the scores they came from, as the A operand of the second products;
// X0 and X1 serve as K-major operands of the first products and as MN-major operands of the second from one copy in shared
// memory.  A streamed block that neither half of the item's rows keeps is not fetched: of a mask of 64-token blocks that keeps
// 13 % of them, partly at random, query items run 17 % of the pairs, key items 21 %; in tiles of 128 x 128 it would be 25 %.
// Roles: warp 0 TMA producer, 1 and 3 MMA issuers, 2 tensor-memory allocation, 3 first the item's block list, 4 and up
// elementwise.
//
// Measured (B200): three heads of 115,456 tokens, block 128, 15 % kept, D = 128 8.6 - 8.8 ms a call in a loop of calls = 0.91 -
// 0.93 PFLOP/s on the five products of the kept pairs (55 - 56 % of the measured burst rate; 1.27 - 1.3 PFLOP/s on the seven that
// run, 90 - 92 % of what a library product sustains); a few launches after a pause, before the clocks fall to 1.6 GHz at the power
// limit, 7.4 - 7.5 ms.  Dense 24 x 4,096 545 us; six heads of 45,104, block 64, D = 64 1.78 ms after a pause, 2.04 - 2.09 in a
// loop.  ncu, eight heads of 16,640 tokens at 25 %: tensor pipe 71 % at D = 128, 55 %
// at D = 64, exponential unit 41 and 43 %.  What bounds it: at D = 128 power and the tensor pipe; at D = 64 the chain of waits
// that a 64-column step is (scores, probabilities, dP, dS, products), of which tensor memory has room for three at a time.
// From the first working version (one step at a time, 8 elementwise warps, 128-row tiles) 9.95 ms, 689 us and 4.36 ms.
//
// Sums are float32 in tensor memory; P and dS are rounded to the inputs' type once, for the second products.  P <= 1 falls
// with the number of keys: for float16 it is held 2^8 times larger (its normal range then reaches 2^-22) and the factor is
// taken out of dS before its rounding and of dV at the end.  dS keeps its natural size.  Held 2^8 larger as well it would be finer
// for small gradients over many keys (17,000 keys: dq off by 0.8 % at a dout of 0.002, 0.08 % at 0.02, 0.02 % at 1), but it would
// overflow past 255, which it reaches at a dout of 64 over four keys (768 there, 13,700 at 1,024) where all results are in range.
// A scaled loss, which float16 training has anyway, moves dS up together with the results and leaves their range to them.
// Every wait is bounded (ptx::mbar_wait) and reports as in the forward.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace moddit {
namespace {

constexpr int kCols = 32;              // streamed columns of a thread
// 4 control warps, then warpgroups of elementwise work
template <int D>
constexpr int kThreads = D == 64 ? 512 : 640;
constexpr int kTile = 128;             // rows of a work item
constexpr int kBlock = 64;             // streamed rows that are kept or left out together
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHalfShift = 8.f;      // float16: P is held 2^kHalfShift times larger
constexpr int kLongKeys = 2, kLongQueries = 4;      // items of every head that start first (the order lists put long ones there)

struct Lists {
  const int32_t *counts, *entries, *order;
};

struct BwdArgs {
  Lists key_lists, query_lists;       // of the key items (by key tile) and of the query items (by pair of query tiles)
  const void *q, *k, *v, *dout;
  const float* nlse;                  // (BH, npad): -lse * log2 e (+ kHalfShift), -inf for rows that attend to nothing
  const float* ndelta;                // (BH, npad): -delta (* 2^-kHalfShift)
  void *dq, *dk, *dv;
  int32_t* status;
  int Hm, batches, N, ntiles, npad, q_split, kvl_lo, kvl_hi;
  float scale, scale_log2;
};

// Which work item a block has: `keys`, position in the kind's start order and batch.  The longest items of every head and
// batch come first, then batch after batch the key items and the (shorter) query items.
struct Item {
  bool keys;
  int pos, batch;
};
__device__ __forceinline__ Item item_of(const BwdArgs& a) {
  const int n_keys = a.ntiles * a.Hm, n_queries = (a.ntiles + (a.ntiles & 1)) * a.Hm;
  const int lk = min(n_keys, kLongKeys * a.Hm), lq = min(n_queries, kLongQueries * a.Hm);
  const int first = (lk + lq) * a.batches;
  int b = static_cast<int>(blockIdx.x);
  Item it;
  if (b < first) {
    const int p = b / a.batches;
    it.batch = b - p * a.batches;
    it.keys = p < lk;
    it.pos = it.keys ? p : p - lk;
  } else {
    b -= first;
    const int rest = n_keys - lk + n_queries - lq;
    it.batch = b / rest;
    const int p = b - it.batch * rest;
    it.keys = p < n_keys - lk;
    it.pos = it.keys ? lk + p : lq + p - (n_keys - lk);
  }
  return it;
}

// The streamed 64-row blocks of a work item, in list order, as (first row << 2) | halves: bit i of `halves` says that rows
// [64 i, 64 i + 64) of the item keep the block.  A list entry names a streamed tile of 128 rows and its kept quarters; blocks
// that start at or past `limit` are left out.  One warp writes them to shared memory and returns how many there are.
// The first entries are asked for together with the count (a list has room for `room`).
template <bool kKeys>
__device__ __forceinline__ int expand(const int32_t* ent, const int32_t* counts, int room, int shift, int limit, int32_t* blocks) {
  const int lane = threadIdx.x % 32;
  int en_next = lane < room ? __ldg(ent + lane) : 0;
  const int count = __ldg(counts);
  int n = 0;
  for (int e0 = 0; e0 < count; e0 += 32) {
    const int en = en_next;
    en_next = e0 + 32 + lane < count ? __ldg(ent + e0 + 32 + lane) : 0;
    const int fl = en >> shift, x0 = (en >> 8) * kTile;
    int bits[2];
    for (int half = 0; half < 2; ++half) {
      bits[half] = kKeys ? (fl >> (2 * half)) & 3 : ((fl >> half) & 1) | ((fl >> (1 + half)) & 2);
      if (e0 + lane >= count || x0 + kBlock * half >= limit) bits[half] = 0;
    }
    const unsigned lo = __ballot_sync(0xffffffffu, bits[0] != 0), hi = __ballot_sync(0xffffffffu, bits[1] != 0);
    const unsigned below = (1u << lane) - 1;
    const int at = n + __popc(lo & below) + __popc(hi & below);
    if (bits[0]) blocks[at] = (x0 << 2) | bits[0];
    if (bits[1]) blocks[at + (bits[0] != 0)] = ((x0 + kBlock) << 2) | bits[1];
    n += __popc(lo) + __popc(hi);
  }
  return n;
}

// Where the limits end in different blocks: leaves out of a list of `expand` the halves, and the blocks, in which no query may see a key, so that
// what such rows hold is never multiplied.  A function of its own, called there only: inside `expand` it changed what the compiler
// made of the rest (query items at D = 128 177 -> 183 us); like this nothing is slower.
__device__ __noinline__ int visible(const BwdArgs& a, bool keys, int row0, int n, int32_t* blocks) {
  const int lane = threadIdx.x % 32;
  int kept = 0;
  __syncwarp();
  for (int i = 0; i < n; i += 32) {
    int32_t block = i + lane < n ? blocks[i + lane] : 0;
    for (int half = 0; half < 2; ++half) {
      const int q0 = keys ? block >> 2 : row0 + kBlock * half, k0 = keys ? row0 + kBlock * half : block >> 2;
      if (k0 >= (q0 + kBlock <= a.q_split ? a.kvl_lo : q0 >= a.q_split ? a.kvl_hi : max(a.kvl_lo, a.kvl_hi))) block &= ~(1 << half);
    }
    const unsigned left = __ballot_sync(0xffffffffu, (block & 3) != 0);
    __syncwarp();
    if (block & 3) blocks[kept + __popc(left & ((1u << lane) - 1))] = block;
    __syncwarp();
    kept += __popc(left);
  }
  return kept;
}

__device__ __forceinline__ void report(int32_t* status, int code, int role, int where) {
  if (atomicCAS(status, 0, code) == 0) {
    status[1] = static_cast<int32_t>(blockIdx.x);
    status[2] = role;
    status[3] = where;
  }
}

template <bool kBF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kBF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// dP - delta for a pair of values (float16: both 2^-kHalfShift times, which undoes the factor that P carries)
template <bool kBF16>
__device__ __forceinline__ uint64_t minus_delta(uint64_t dp, uint64_t nd) {
  if constexpr (kBF16) return ptx::add_f32x2(dp, nd);
  const float down = 1.f / 256.f;
  return ptx::fma_f32x2(dp, ptx::pack_f32x2(down, down), nd);
}

// ---------------------------------------------------------------------------------------------------------------
// Elementwise work on kCols columns: P = 2^(S scale + nlse) and dS = P (dP - delta).  P and dS are packed over the first half
// of the columns that they come from.
//
// Query items: a thread has one row, so the row's statistics are two registers.
template <bool kBF16>
struct QueryRows {
  float p[kCols];
  __device__ __forceinline__ void load(uint32_t tS) {
    ptx::tmem_ld32(tS, reinterpret_cast<uint32_t*>(p));
    ptx::tmem_ld_wait();
  }
  __device__ __forceinline__ void probabilities(uint64_t scale2, float nl, int below) {      // columns >= below are masked
    const uint64_t nl2 = ptx::pack_f32x2(nl, nl);
#pragma unroll
    for (int i = 0; i < kCols / 2; ++i) {
      float x0, x1;
      ptx::unpack_f32x2(ptx::fma_f32x2(ptx::pack_f32x2(p[2 * i], p[2 * i + 1]), scale2, nl2), x0, x1);
      p[2 * i] = ptx::ex2(x0);
      p[2 * i + 1] = ptx::ex2(x1);
    }
    if (__any_sync(0xffffffffu, below < kCols)) {
#pragma unroll
      for (int c = 0; c < kCols; ++c) p[c] = c < below ? p[c] : 0.f;
    }
  }
  // reads dP, stores dS over it
  __device__ __forceinline__ void scores_gradient(uint32_t tP, float nd, int below) {
    const uint64_t nd2 = ptx::pack_f32x2(nd, nd);
    const bool masked = __any_sync(0xffffffffu, below < kCols);
    float d[kCols];
    ptx::tmem_ld32(tP, reinterpret_cast<uint32_t*>(d));
    ptx::tmem_ld_wait();
    if (masked) {                     // what lies in a masked place may be anything
#pragma unroll
      for (int c = 0; c < kCols; ++c) d[c] = c < below ? d[c] : 0.f;
    }
    uint32_t pk[kCols / 2];
#pragma unroll
    for (int i = 0; i < kCols / 2; ++i) {
      const uint64_t t = ptx::mul_f32x2(minus_delta<kBF16>(ptx::pack_f32x2(d[2 * i], d[2 * i + 1]), nd2),
                                        ptx::pack_f32x2(p[2 * i], p[2 * i + 1]));
      float y0, y1;
      ptx::unpack_f32x2(t, y0, y1);
      pk[i] = pack2<kBF16>(y0, y1);
    }
    ptx::tmem_st16(tP, pk);
  }
};

// Key items: columns are queries, so every column has statistics of its own.  A thread has four rows and eight columns
// (fragments of tcgen05.ld.16x256b): it reads 8 column statistics from shared memory for 32 values.  With one row and 32
// columns a thread it would read all 32, a warp-wide shared-memory access each - as many cycles of the shared memory as the
// products of a tile take from it.
template <bool kBF16>
struct KeyRows {
  float p[2][16];
  // which places are masked: rows by `lo`, `hi` (bit j: row i / 4 + 8 j may see queries before / from column `split` on)
  struct Mask {
    bool on;
    int split, lo, hi;
  };
  // zeros in the masked places of column groups [g0, g1)
  __device__ __forceinline__ void clear(float (&v)[2][16], const Mask& m, int g0, int g1) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (g < g0 || g >= g1) continue;
        const int rows = 8 * g + 2 * static_cast<int>(threadIdx.x % 4) + i < m.split ? m.lo : m.hi;
#pragma unroll
        for (int row = 0; row < 4; ++row) {
          float& x = v[row >> 1][4 * g + 2 * (row & 1) + i];
          x = ((rows >> row) & 1) ? x : 0.f;
        }
      }
  }
  __device__ __forceinline__ void load(uint32_t tS) {
    ptx::tmem_ld_16x32(tS, reinterpret_cast<uint32_t*>(p[0]));
    ptx::tmem_ld_16x32(tS + (16u << 16), reinterpret_cast<uint32_t*>(p[1]));
    ptx::tmem_ld_wait();
  }
  // f(half of the lanes, pair of values, column group) over all pairs of a thread
  template <class F>
  __device__ __forceinline__ void pairs(F&& f) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int lh = 0; lh < 2; ++lh)
#pragma unroll
        for (int j = 0; j < 2; ++j) f(lh, 2 * g + j, g);
  }
  // P of column groups [kG0, kG0 + kGs), stored over the first half of the columns of S
  template <int kG0, int kGs>
  __device__ __forceinline__ void probabilities(uint32_t tS, uint64_t scale2, const float* nl, const Mask& m) {
#pragma unroll
    for (int g = kG0; g < kG0 + kGs; ++g) {
      const uint64_t nl2 = *reinterpret_cast<const uint64_t*>(nl + 8 * g + 2 * (threadIdx.x % 4));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float* v = p[i >> 1] + 4 * g + 2 * (i & 1);
        float x0, x1;
        ptx::unpack_f32x2(ptx::fma_f32x2(ptx::pack_f32x2(v[0], v[1]), scale2, nl2), x0, x1);
        v[0] = ptx::ex2(x0);
        v[1] = ptx::ex2(x1);
      }
    }
    if (m.on) clear(p, m, kG0, kG0 + kGs);
    uint32_t pk[2][2 * kGs];
#pragma unroll
    for (int g = kG0; g < kG0 + kGs; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* v = p[i >> 1] + 4 * g + 2 * (i & 1);
        pk[i >> 1][2 * (g - kG0) + (i & 1)] = pack2<kBF16>(v[0], v[1]);
      }
#pragma unroll
    for (int lh = 0; lh < 2; ++lh) {
      const uint32_t to = tS + (static_cast<uint32_t>(16 * lh) << 16) + 4 * kG0;
      if constexpr (kGs == 4) ptx::tmem_st_16x4g(to, pk[lh]);
      else ptx::tmem_st_16x2g(to, pk[lh]);
    }
  }
  __device__ __forceinline__ void scores_gradient(uint32_t tP, const float* nd, const Mask& m) {
    uint64_t nd2[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) nd2[g] = *reinterpret_cast<const uint64_t*>(nd + 8 * g + 2 * (threadIdx.x % 4));
    float d[2][16];
    ptx::tmem_ld_16x32(tP, reinterpret_cast<uint32_t*>(d[0]));
    ptx::tmem_ld_16x32(tP + (16u << 16), reinterpret_cast<uint32_t*>(d[1]));
    ptx::tmem_ld_wait();
    if (m.on) clear(d, m, 0, 4);         // what lies in a masked place may be anything
    uint32_t pk[2][8];
    pairs([&](int lh, int i, int g) {
      const uint64_t t = ptx::mul_f32x2(minus_delta<kBF16>(ptx::pack_f32x2(d[lh][2 * i], d[lh][2 * i + 1]), nd2[g]),
                                        ptx::pack_f32x2(p[lh][2 * i], p[lh][2 * i + 1]));
      float y0, y1;
      ptx::unpack_f32x2(t, y0, y1);
      pk[lh][i] = pack2<kBF16>(y0, y1);
    });
    ptx::tmem_st_16x4g(tP, pk[0]);
    ptx::tmem_st_16x4g(tP + (16u << 16), pk[1]);
  }
};

// Packed zeros (P or dS of rows that keep nothing of a block)
__device__ __forceinline__ void store_zeros(uint32_t t) {
  uint32_t z[kCols / 2];
#pragma unroll
  for (int i = 0; i < kCols / 2; ++i) z[i] = 0u;
  ptx::tmem_st16(t, z);
}

__device__ __forceinline__ void hand_over(uint32_t bar) {
  ptx::tmem_st_wait();
  ptx::tc_fence_before();
  __syncwarp();
  if (threadIdx.x % 32 == 0) ptx::mbar_arrive(bar);
}

// kWidth accumulator columns of this thread's row, times f, as 16-bit values to dst; zeros where nothing was accumulated
template <bool kBF16, int kWidth>
__device__ __forceinline__ void store_rows(uint32_t t, bool any, bool in, float f, uint4* dst) {
  float o[kWidth];
  if (any) {
    if constexpr (kWidth == 32) ptx::tmem_ld32(t, reinterpret_cast<uint32_t*>(o));
    else ptx::tmem_ld16(t, reinterpret_cast<uint32_t*>(o));
    ptx::tmem_ld_wait();
  } else {
#pragma unroll
    for (int i = 0; i < kWidth; ++i) o[i] = 0.f;
  }
  if (!in) return;
#pragma unroll
  for (int i = 0; i < kWidth / 8; ++i) {
    uint4 w;
    w.x = pack2<kBF16>(o[i * 8 + 0] * f, o[i * 8 + 1] * f);
    w.y = pack2<kBF16>(o[i * 8 + 2] * f, o[i * 8 + 3] * f);
    w.z = pack2<kBF16>(o[i * 8 + 4] * f, o[i * 8 + 5] * f);
    w.w = pack2<kBF16>(o[i * 8 + 6] * f, o[i * 8 + 7] * f);
    dst[i] = w;
  }
}

// What an elementwise thread of a query item reads while the block is set up: 32 words of a row of Q or dO (which end up in
// tensor memory; at D = 64 two warpgroups have a row each, at D = 128 four half a row), zeros past the last row.  Not the row's
// statistics: the kernel that computes them may still be at work then.
template <int D>
struct Fixed {
  uint32_t v[32];
  static __device__ __forceinline__ int group() { return (static_cast<int>(threadIdx.x) - 128) / 128; }
  static __device__ __forceinline__ int which() { return D == 64 ? group() : group() / 2; }
  static __device__ __forceinline__ int part() { return D == 64 ? 0 : group() & 1; }
  static __device__ __forceinline__ bool mine() { return which() < 2; }
  __device__ __forceinline__ void load(const BwdArgs& a, int bh, int row0) {
    if (!mine()) return;
    const int grow = row0 + threadIdx.x % 128;
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(which() ? a.dout : a.q) +
                                                      (static_cast<int64_t>(bh) * a.N + grow) * D * 2) + part() * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 x = grow < a.N ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
      v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
    }
  }
};

struct Block {                        // what all roles of a block know
  unsigned char* smem;                // 1024-byte aligned
  uint32_t tmem;
  volatile int* abort_flag;
  uint32_t bar0;
  int row0, bh, count;                // count: streamed blocks
  const int32_t* blocks;              // of `expand`
  __device__ __forceinline__ uint32_t bar(int i) const { return bar0 + 8u * static_cast<uint32_t>(i); }
};

// Waits for a barrier's phase; most are complete when they are asked for (a complete one costs an issuing thread about 100 clocks
// through try_wait).
__device__ __forceinline__ bool await(const Block& b, const BwdArgs& a, int role, int bar, uint32_t parity, int code, int k) {
  if (ptx::mbar_test(b.bar(bar), parity) || ptx::mbar_wait(b.bar(bar), parity, b.abort_flag)) return true;
  report(a.status, code, role, k);
  return false;
}

__device__ __forceinline__ uint64_t advance(uint64_t desc, uint32_t bytes) {
  // the start-address field (bits 0-13, units of 16 bytes) never carries out for shared-memory addresses
  return (desc & 0xffffffff00000000ull) | static_cast<uint32_t>(static_cast<uint32_t>(desc) + (bytes >> 4));
}

constexpr int kMaxStages = 8;
constexpr int kNumBarriers = 2 * kMaxStages + 18;
constexpr int kMaxBlocks = 7168;       // streamed blocks of a work item: 458,752 rows
struct __align__(16) Control {
  float stats[kMaxStages][2][kBlock]; // key items: -lse * log2 e and -delta of the streamed query rows
  unsigned long long bars[kNumBarriers];
  uint32_t tmem_base;
  int abort_flag;
  int count;
  int32_t blocks[kMaxBlocks + 4];       // read ahead past the end
};

// bytes of tiles in shared memory; behind them the control block, before them up to 1024 bytes of alignment
template <int D>
constexpr size_t kTilesBytes = static_cast<size_t>(D == 128 ? 192 : 160) * 1024;

// ---------------------------------------------------------------------------------------------------------------
// Chains: warpgroups of their own take every kC-th streamed block through scores, dP and dS of its own, a part of a step behind
// the other chains, so that some have exponentials to do while the others wait or pack.
//   D = 128 (query items)  two chains of two warpgroups, 32 columns a thread
//   D = 64                 three chains of one warpgroup, 64 columns a thread: the waits and the latencies of a step are bound
//                          here, not a unit, and a third chain hides more of them than a second warpgroup of a chain.
// Fixed tiles live in tensor memory as A operands where there is room (query items), which halves what the first products read
// from shared memory.
// Tensor memory: S_c [64 c, 64 c + 64), then dP_c likewise, then the accumulators and F0, F1.
template <int D, bool kBF16, bool kKeys>
struct Chains {
  static constexpr int kC = D == 64 ? 3 : 2;            // chains
  static constexpr int kG = D == 64 ? 1 : 2;            // warpgroups of a chain
  static constexpr int kU = 2 / kG;                     // units of kCols columns of a thread
  static constexpr int kStages = D == 128 ? 6 : 8;
  static constexpr int kBlockBytes = kBlock * D * 2;
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kChunks = D / 64;
  static constexpr int kChunkBytes = kBlock * 128;
  static constexpr int kStagesAt = kKeys ? 2 * kTileBytes : 0;
  static constexpr int kDP = 64 * kC, kAcc0 = 128 * kC, kAcc1 = kAcc0 + 64, kF = kAcc0 + D;
  static_assert(!kKeys || D == 64, "tensor memory holds two accumulators at D = 64 only");
  static_assert((kKeys ? kAcc1 + 64 : kF + D) <= 512, "tensor memory");
  static_assert(kStagesAt + 2 * kStages * kBlockBytes <= static_cast<int>(kTilesBytes<D>), "shared memory");
  enum { kFixed = 0, kSFull = 1, kDPFull = kSFull + kC, kPDone = kDPFull + kC, kDSDone = kPDone + kC, kDPFree = kDSDone + kC,
         kFinal = kDPFree + kC, kFull, kEmpty = kFull + kStages, kUsed = kEmpty + kStages };
  static_assert(static_cast<int>(kUsed) <= kNumBarriers, "barriers");

  static __device__ __forceinline__ int arrivals(int i) {               // one per warp, copy or commit
    if (i == kFixed) return kKeys ? 1 : D == 64 ? 8 : 16;
    if (i >= kPDone && i < kDPFree) return 4 * kG;
    return kKeys && (i == kFinal || i >= kEmpty) ? 2 : 1;               // key items: of both issuing threads
  }
  // A block's stage and chain and the phases of their barriers, counted along: the issuing threads share their schedulers with
  // busy warps, so every instruction between two products shows.
  struct Place {
    int s = 0, c = 0;
    uint32_t stage_phase = 0, chain_phase = 0;
    __device__ __forceinline__ void next() {
      if (++s == kStages) { s = 0; stage_phase ^= 1; }
      if (++c == kC) { c = 0; chain_phase ^= 1; }
    }
  };

  static __device__ __forceinline__ void produce(const Block& b, const BwdArgs& a, const Control* ctl, const CUtensorMap* tf0,
                                                 const CUtensorMap* tf1, const CUtensorMap* tx0, const CUtensorMap* tx1) {
    if (b.count == 0) return;
    const uint32_t sF = ptx::smem_u32(b.smem), sX = sF + kStagesAt;
    if (kKeys) {
      ptx::mbar_expect_tx(b.bar(kFixed), 2 * kTileBytes);
      for (int h = 0; h < 2; ++h) {
        ptx::tma_load_3d(sF + h * kBlockBytes, tf0, b.bar(kFixed), 0, b.row0 + h * kBlock, b.bh);
        ptx::tma_load_3d(sF + kTileBytes + h * kBlockBytes, tf1, b.bar(kFixed), 0, b.row0 + h * kBlock, b.bh);
      }
    }
    bool ok = true;
    int k = 0;
    for (; k < b.count; ++k) {
      const int s = k % kStages, x0 = b.blocks[k] >> 2;
      ok = ptx::mbar_wait(b.bar(kEmpty + s), ((k / kStages) & 1) ^ 1, b.abort_flag);
      if (!ok) { report(a.status, 1, 0, k); break; }
      const uint32_t to = sX + 2 * s * kBlockBytes;
      ptx::mbar_expect_tx(b.bar(kFull + s), 2 * kBlockBytes + (kKeys ? 2 * kBlock * 4 : 0));
      for (int c = 0; c < kChunks; ++c) {
        ptx::tma_load_3d(to + c * kChunkBytes, tx0, b.bar(kFull + s), c * 64, x0, b.bh);
        ptx::tma_load_3d(to + kBlockBytes + c * kChunkBytes, tx1, b.bar(kFull + s), c * 64, x0, b.bh);
      }
      if (kKeys) {
        const int64_t at = static_cast<int64_t>(b.bh) * a.npad + x0;
        ptx::bulk_load(ptx::smem_u32(ctl->stats[s][0]), a.nlse + at, kBlock * 4, b.bar(kFull + s));
        ptx::bulk_load(ptx::smem_u32(ctl->stats[s][1]), a.ndelta + at, kBlock * 4, b.bar(kFull + s));
      }
    }
    if (!ok) {      // give copies in flight a bounded time to land (their barriers may never be consumed)
      if (kKeys)
        for (int i = 0; i < 4096 && !ptx::mbar_try_wait(b.bar(kFixed), 0); ++i) {}
      for (int m = max(0, k - kStages); m < k; ++m)
        for (int i = 0; i < 4096 && !ptx::mbar_try_wait(b.bar(kFull + m % kStages), (m / kStages) & 1); ++i) {}
    }
  }

  // The products of a block.  which = 0: S = F0 X0^T, 1: dP = F1 X1^T
  static __device__ __forceinline__ void first(const Block& b, int which, const Place& p) {
    constexpr uint32_t kIdesc = ptx::idesc_f16(128, kBlock, kBF16, false);
    const uint32_t sF = ptx::smem_u32(b.smem);
    const uint64_t b0 = advance(ptx::smem_desc_sw128(sF + kStagesAt + which * kBlockBytes, 16, 1024), 2 * p.s * kBlockBytes);
    const uint64_t a0 = ptx::smem_desc_sw128(sF + which * kTileBytes, 16, 1024);      // both K-major
    const uint32_t d = b.tmem + which * kDP + p.c * 64;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const uint64_t bk = advance(b0, (kk / 4) * kChunkBytes + (kk % 4) * 32);
      if constexpr (kKeys) ptx::mma_ss(d, advance(a0, kk * 32), bk, kIdesc, kk > 0 ? 1u : 0u);
      else ptx::mma_ts(d, b.tmem + kF + which * (D / 2) + kk * 8, bk, kIdesc, kk > 0 ? 1u : 0u);
    }
    ptx::tc_commit(b.bar((which ? kDPFull : kSFull) + p.c));
  }
  // which = 0: acc1 += P X1, 1: acc0 += dS X0; acc: whether there is anything in the accumulator yet
  static __device__ __forceinline__ void second(const Block& b, int which, const Place& p, uint32_t acc) {
    constexpr uint32_t kIdesc = ptx::idesc_f16(128, D, kBF16, true);
    const uint64_t b0 = advance(ptx::smem_desc_sw128(ptx::smem_u32(b.smem) + kStagesAt + (1 - which) * kBlockBytes, kChunkBytes, 1024),
                                2 * p.s * kBlockBytes);       // MN-major
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      ptx::mma_ts(b.tmem + (which ? kAcc0 : kAcc1), b.tmem + which * kDP + p.c * 64 + (kk >> 1) * 32 + (kk & 1) * 8,
                  advance(b0, kk * 2048), kIdesc, kk > 0 ? 1u : acc);
  }

  static __device__ __forceinline__ bool landed(const Block& b, const BwdArgs& a, int role, const Place& p, int k) {
    return await(b, a, role, kFull + p.s, p.stage_phase, 2, k);
  }
  // for what the elementwise warps have read from or written to tensor memory
  static __device__ __forceinline__ bool wait(const Block& b, const BwdArgs& a, int role, int bar, uint32_t parity, int code, int k) {
    const bool ok = await(b, a, role, bar, parity, code, k);
    ptx::tc_fence_after();
    return ok;
  }

  // Two issuing threads.  Products of one thread run in the order of issue; a thread hands over an instruction about every 30
  // clocks, spends up to 100 on a wait and shares its scheduler with busy warps, so one for everything is the bound.
  // By sides: thread 0 has acc1 += P(k) X1 (key items) and S(k + kC), which overwrites that P; thread 1 has acc0 += dS(k) X0 and
  // dP(k + kC), which overwrites that dS.  No column of tensor memory is shared.
  // By kinds (query items at D = 64): thread 0 has the first products, thread 1 the second; dP(k + kC) then waits for the
  // completion of dS(k) X0, but thread 0 fills both buffers as soon as either is free.
  // Dense 18,944 rows alone, all by one thread / by sides / by kinds: key items at D = 64 171 / 167 / 193 us, query items at
  // D = 64 160 / 158 / 147, at D = 128 201 / 183 / 189; key items at D = 128 (Pairs) 264 / 280 / -.  A third thread for dP alone:
  // 156 and 199.
  static __device__ __forceinline__ void issue_side(const Block& b, const BwdArgs& a, int side) {
    const int role = side ? 6 : 1;
    Place here, ahead;                // of blocks k and k + kC
    bool ok = b.count == 0 || wait(b, a, role, kFixed, 0, 2, -1);
    for (int k = 0; k < min(kC, b.count) && ok; ++k, ahead.next()) {
      ok = landed(b, a, role, ahead, k);
      if (ok) first(b, side, ahead);
    }
    for (int k = 0; k < b.count && ok; ++k, here.next(), ahead.next()) {
      if (!wait(b, a, role, (side ? kDSDone : kPDone) + here.c, here.chain_phase, 3, k)) break;
      if (kKeys || side) {
        second(b, side, here, k > 0);
        ptx::tc_commit(b.bar(kEmpty + here.s));
      }
      if (k + kC < b.count) {
        if (!landed(b, a, role, ahead, k + kC)) break;
        first(b, side, ahead);
      }
    }
    if (kKeys || side) ptx::tc_commit(b.bar(kFinal));
  }

  static __device__ __forceinline__ void issue_kind(const Block& b, const BwdArgs& a, int kind) {
    if (kind == 0) {
      // a chain's barriers are in the other phase of its last block
      if (b.count == 0 || !wait(b, a, 1, kFixed, 0, 2, -1)) return;
      Place here, behind;             // blocks k and k - 1
      for (int k = 0; k <= b.count; ++k) {
        if (k < b.count) {
          if (k >= kC && !wait(b, a, 1, kPDone + here.c, here.chain_phase ^ 1, 3, k)) return;
          if (!landed(b, a, 1, here, k)) return;
          first(b, 0, here);
          here.next();
        }
        if (k >= 1) {
          if (k - 1 >= kC && !wait(b, a, 1, kDPFree + behind.c, behind.chain_phase ^ 1, 4, k)) return;
          first(b, 1, behind);
          behind.next();
        }
      }
    } else {
      Place here;
      for (int k = 0; k < b.count; ++k, here.next()) {
        if (!landed(b, a, 6, here, k) || !wait(b, a, 6, kDSDone + here.c, here.chain_phase, 4, k)) break;
        second(b, 1, here, k > 0);
        ptx::tc_commit(b.bar(kDPFree + here.c));
        ptx::tc_commit(b.bar(kEmpty + here.s));
      }
      ptx::tc_commit(b.bar(kFinal));
    }
  }

  static __device__ __forceinline__ void issue(const Block& b, const BwdArgs& a, int thread) {
    if constexpr (!kKeys && D == 64) issue_kind(b, a, thread);
    else issue_side(b, a, thread);
  }

  static __device__ __forceinline__ void compute(const Block& b, const BwdArgs& a, const Control* ctl, const Fixed<D>& fixed, int warp,
                                                 int lane) {
    const int wg = (warp - 4) / 4;
    const int c = wg / kG;                        // chain
    const int u0 = wg % kG;                       // first unit of this thread
    const int wq = warp % 4;                      // tensor-memory lane quarter
    const int grow = b.row0 + wq * 32 + lane;
    const uint32_t t = b.tmem + (static_cast<uint32_t>(wq * 32) << 16);
    const uint32_t tS = t + c * 64 + u0 * kCols, tP = tS + kDP;
    const int kv_min = min(a.kvl_lo, a.kvl_hi);
    if (!kKeys && fixed.mine()) {
      ptx::tmem_st32(t + kF + fixed.which() * (D / 2) + fixed.part() * 32, fixed.v);
      hand_over(b.bar(kFixed));
    }
    float nl = 0.f, nd = 0.f;                     // query items: the row's statistics, which are there since the wait for them
    if (!kKeys) {
      const int64_t at = static_cast<int64_t>(b.bh) * a.npad + grow;
      nl = a.nlse[at];
      nd = a.ndelta[at];
    }
    const int lim = grow < a.q_split ? a.kvl_lo : a.kvl_hi;
    int rows_lo = 0, rows_hi = 0;                 // key items: which of this thread's four rows lie below the limits
    if (kKeys)
      for (int j = 0; j < 4; ++j) {
        const int key = b.row0 + wq * 32 + 8 * j + lane / 4;
        rows_lo |= (key < a.kvl_lo) << j;
        rows_hi |= (key < a.kvl_hi) << j;
      }
    const uint64_t scale2 = ptx::pack_f32x2(a.scale_log2, a.scale_log2);
    bool ok = true;
    auto wait_all = [&](int bar, uint32_t parity, int code, int k) {
      ok = __all_sync(0xffffffffu, ptx::mbar_wait(b.bar(bar), parity, b.abort_flag));
      if (!ok && lane == 0) report(a.status, code, 2 + c, k);
      ptx::tc_fence_after();
      return ok;
    };
    int next = b.blocks[c];           // read ahead; past the end it is not used
    uint32_t par = 0;
    for (int k = c; k < b.count; k += kC, par ^= 1) {
      const int x0 = next >> 2, bits = next & 3;
      next = b.blocks[k + kC];
      const int s = k % kStages;
      if (!wait_all(kSFull + c, par, 5, k)) break;      // the statistics came with the operands
      if (!((bits >> (wq >> 1)) & 1)) {           // these rows keep nothing of the block
        if (kKeys)
          for (int u = 0; u < kU; ++u) store_zeros(tS + u * kCols);
        hand_over(b.bar(kPDone + c));
        if (!wait_all(kDPFull + c, par, 6, k)) break;
        for (int u = 0; u < kU; ++u) store_zeros(tP + u * kCols);
        hand_over(b.bar(kDSDone + c));
        continue;
      }
      if constexpr (kKeys) {
        KeyRows<kBF16> x[kU];
        const float* stats = ctl->stats[s][0] + u0 * kCols;
        typename KeyRows<kBF16>::Mask m{b.row0 + kTile > kv_min, a.q_split - x0 - u0 * kCols, rows_lo, rows_hi};
#pragma unroll
        for (int u = 0; u < kU; ++u) x[u].load(tS + u * kCols);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          x[u].template probabilities<0, 4>(tS + u * kCols, scale2, stats + u * kCols, m);
          m.split -= kCols;
        }
        hand_over(b.bar(kPDone + c));
        if (!wait_all(kDPFull + c, par, 6, k)) break;
        m.split += kU * kCols;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          x[u].scores_gradient(tP + u * kCols, stats + kBlock + u * kCols, m);
          m.split -= kCols;
        }
      } else {
        QueryRows<kBF16> x[kU];
        const int below = lim - x0 - u0 * kCols;
#pragma unroll
        for (int u = 0; u < kU; ++u) x[u].load(tS + u * kCols);
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(b.bar(kPDone + c));      // P stays in registers: the next scores may overwrite these
#pragma unroll
        for (int u = 0; u < kU; ++u) x[u].probabilities(scale2, nl, below - u * kCols);
        if (!wait_all(kDPFull + c, par, 6, k)) break;
#pragma unroll
        for (int u = 0; u < kU; ++u) x[u].scores_gradient(tP + u * kCols, nd, below - u * kCols);
      }
      hand_over(b.bar(kDSDone + c));
    }
    if (!ok || !wait_all(kFinal, 0, 7, -1)) return;
    // 32 columns of an accumulator at a time for each warpgroup
    for (int unit = wg; unit < (kKeys ? 2 : 1) * (D / 32); unit += kC * kG) {
      const int which = unit / (D / 32), col = unit % (D / 32) * 32;
      const int64_t at = ((static_cast<int64_t>(b.bh) * a.N + grow) * D + col) * 2;
      store_rows<kBF16, 32>(t + (which ? kAcc1 : kAcc0) + col, b.count > 0, grow < a.N, which ? (kBF16 ? 1.f : exp2f(-kHalfShift)) : a.scale,
                            reinterpret_cast<uint4*>(static_cast<unsigned char*>(which ? a.dv : kKeys ? a.dk : a.dq) + at));
    }
  }
};

// ---------------------------------------------------------------------------------------------------------------
// Key items at D = 128: the four 128-column regions fill tensor memory, so the fixed tiles stay in shared memory and both
// warpgroups work on one pair of streamed blocks.  A product with both operands in shared memory reads it at its full rate,
// and at N = 64 it would take 52 clocks of the pipe for 32 of work: hence 128 columns at a time.
// Tensor memory: S [0, 128) dP [128, 256) acc0 [256, 384) acc1 [384, 512).
template <bool kBF16>
struct Pairs {
  static constexpr int D = 128;
  static constexpr int kStages = 2;
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kChunkBytes = kTile * 128;
  static constexpr int kHalfBytes = kBlock * 128;       // a block's rows of one 64-element chunk
  enum { kFixed = 0, kSFull, kDPFull, kPLo, kPHi, kDSDone, kFinal, kFull, kEmpty = kFull + kStages, kUsed = kEmpty + kStages };

  static __device__ __forceinline__ int arrivals(int i) { return (i >= kPLo && i <= kDSDone) ? 16 : 1; }

  static __device__ __forceinline__ void produce(const Block& b, const BwdArgs& a, const Control* ctl, const CUtensorMap* tf0,
                                                 const CUtensorMap* tf1, const CUtensorMap* tx0, const CUtensorMap* tx1) {
    const uint32_t sF = ptx::smem_u32(b.smem), sX = sF + 2 * kTileBytes;
    if (b.count == 0) return;
    ptx::mbar_expect_tx(b.bar(kFixed), 2 * kTileBytes);
    for (int c = 0; c < 2; ++c)
      for (int h = 0; h < 2; ++h) {
        const uint32_t to = sF + c * kChunkBytes + h * kHalfBytes;
        ptx::tma_load_3d(to, tf0, b.bar(kFixed), c * 64, b.row0 + h * kBlock, b.bh);
        ptx::tma_load_3d(to + kTileBytes, tf1, b.bar(kFixed), c * 64, b.row0 + h * kBlock, b.bh);
      }
    bool ok = true;
    int n = 0;
    for (; 2 * n < b.count; ++n) {
      const int s = n % kStages;
      ok = ptx::mbar_wait(b.bar(kEmpty + s), ((n / kStages) & 1) ^ 1, b.abort_flag);
      if (!ok) { report(a.status, 1, 0, n); break; }
      ptx::mbar_expect_tx(b.bar(kFull + s), 2 * kTileBytes + 4 * kBlock * 4);
      for (int h = 0; h < 2; ++h) {
        const int x0 = b.blocks[min(2 * n + h, b.count - 1)] >> 2;      // an odd last block is there twice, once masked
        const uint32_t to = sX + 2 * s * kTileBytes + h * kHalfBytes;
        for (int c = 0; c < 2; ++c) {
          ptx::tma_load_3d(to + c * kChunkBytes, tx0, b.bar(kFull + s), c * 64, x0, b.bh);
          ptx::tma_load_3d(to + kTileBytes + c * kChunkBytes, tx1, b.bar(kFull + s), c * 64, x0, b.bh);
        }
        const int64_t at = static_cast<int64_t>(b.bh) * a.npad + x0;
        ptx::bulk_load(ptx::smem_u32(ctl->stats[2 * s + h][0]), a.nlse + at, kBlock * 4, b.bar(kFull + s));
        ptx::bulk_load(ptx::smem_u32(ctl->stats[2 * s + h][1]), a.ndelta + at, kBlock * 4, b.bar(kFull + s));
      }
    }
    if (!ok) {
      for (int i = 0; i < 4096 && !ptx::mbar_try_wait(b.bar(kFixed), 0); ++i) {}
      for (int m = max(0, n - kStages); m < n; ++m)
        for (int i = 0; i < 4096 && !ptx::mbar_try_wait(b.bar(kFull + m % kStages), (m / kStages) & 1); ++i) {}
    }
  }

  static __device__ __forceinline__ void issue(const Block& b, const BwdArgs& a, int thread) {
    if (thread != 0) return;
    constexpr uint32_t kIdescS = ptx::idesc_f16(128, 128, kBF16, false);
    constexpr uint32_t kIdescG = ptx::idesc_f16(128, D, kBF16, true);
    const uint32_t sF = ptx::smem_u32(b.smem), sX = sF + 2 * kTileBytes;
    const uint64_t df = ptx::smem_desc_sw128(sF, 16, 1024);                // K-major: F0, F1 and the X tiles
    const uint64_t dx = advance(df, sX - sF);
    const uint64_t dg = ptx::smem_desc_sw128(sX, kChunkBytes, 1024);       // MN-major: the X tiles
    auto first = [&](int which, int s) {
      const uint64_t a0 = advance(df, which * kTileBytes), b0 = advance(dx, (2 * s + which) * kTileBytes);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t off = (kk / 4) * kChunkBytes + (kk % 4) * 32;
        ptx::mma_ss(b.tmem + which * 128, advance(a0, off), advance(b0, off), kIdescS, kk > 0 ? 1u : 0u);
      }
      ptx::tc_commit(b.bar(kSFull + which));
    };
    // which = 0: acc1 += P X1, 1: acc0 += dS X0, steps kk0, kk0 + by, ... of 16 rows; a warpgroup's 32 columns are two steps
    auto second = [&](int which, int s, uint32_t acc, int kk0, int by) {
      const uint64_t b0 = advance(dg, (2 * s + 1 - which) * kTileBytes);
#pragma unroll
      for (int kk = kk0; kk < 8; kk += by)
        ptx::mma_ts(b.tmem + (which ? 256 : 384), b.tmem + which * 128 + (kk >> 1) * 32 + (kk & 1) * 8, advance(b0, kk * 2048),
                    kIdescG, (acc || kk > kk0) ? 1u : 0u);
    };
    const int steps = (b.count + 1) / 2;
    bool ok = true;
    if (steps > 0) {
      ok = await(b, a, 1, kFixed, 0, 2, -1) && await(b, a, 1, kFull, 0, 2, -1);
      if (ok) { first(0, 0); first(1, 0); }
    }
    for (int n = 0; n < steps && ok; ++n) {
      const int s = n % kStages, s1 = (n + 1) % kStages;
      const bool next = n + 1 < steps;
      if (!await(b, a, 1, kPLo, n & 1, 3, n)) break;
      ptx::tc_fence_after();
      second(0, s, n > 0, 0, 2);
      if (!await(b, a, 1, kPHi, n & 1, 3, n)) break;
      ptx::tc_fence_after();
      second(0, s, 1u, 1, 2);
      if (next) {
        if (!await(b, a, 1, kFull + s1, ((n + 1) / kStages) & 1, 2, n)) break;
        first(0, s1);
      }
      if (!await(b, a, 1, kDSDone, n & 1, 4, n)) break;
      ptx::tc_fence_after();
      second(1, s, n > 0, 0, 1);
      ptx::tc_commit(b.bar(kEmpty + s));
      if (next) first(1, s1);
    }
    ptx::tc_commit(b.bar(kFinal));
  }

  static __device__ __forceinline__ void compute(const Block& b, const BwdArgs& a, const Control* ctl, const Fixed<D>&, int warp,
                                                 int lane) {
    const int h = (warp - 4) / 8;                 // which of the two streamed blocks
    const int u = ((warp - 4) / 4) & 1;           // half of its columns
    const int wq = warp % 4;
    const uint32_t lane_base = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t tS = b.tmem + lane_base + h * 64 + u * kCols, tP = tS + 128;
    const int kv_min = min(a.kvl_lo, a.kvl_hi);
    int rows_lo = 0, rows_hi = 0;
    for (int j = 0; j < 4; ++j) {
      const int key = b.row0 + wq * 32 + 8 * j + lane / 4;
      rows_lo |= (key < a.kvl_lo) << j;
      rows_hi |= (key < a.kvl_hi) << j;
    }
    const uint64_t scale2 = ptx::pack_f32x2(a.scale_log2, a.scale_log2);
    bool ok = true;
    int next = b.blocks[h];           // read ahead; past the end it counts for nothing
    for (int n = 0; 2 * n < b.count; ++n) {
      const int x0 = next >> 2, bits = 2 * n + h < b.count ? next & 3 : 0;
      next = b.blocks[2 * n + 2 + h];
      const int s = n % kStages;
      ok = ptx::mbar_wait(b.bar(kSFull), n & 1, b.abort_flag);      // the statistics came with the operands
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) { if (lane == 0) report(a.status, 5, 2 + h, n); break; }
      ptx::tc_fence_after();
      const bool mine = (bits >> (wq >> 1)) & 1;
      KeyRows<kBF16> x;
      const typename KeyRows<kBF16>::Mask m{b.row0 + kTile > kv_min, a.q_split - x0 - u * kCols, rows_lo, rows_hi};
      if (mine) {
        x.load(tS);
        x.template probabilities<0, 2>(tS, scale2, ctl->stats[2 * s + h][0] + u * kCols, m);
        hand_over(b.bar(kPLo));
        x.template probabilities<2, 2>(tS, scale2, ctl->stats[2 * s + h][0] + u * kCols, m);
      } else {
        store_zeros(tS);
        hand_over(b.bar(kPLo));
      }
      hand_over(b.bar(kPHi));
      ok = __all_sync(0xffffffffu, ptx::mbar_wait(b.bar(kDPFull), n & 1, b.abort_flag));
      if (!ok) { if (lane == 0) report(a.status, 6, 2 + h, n); break; }
      ptx::tc_fence_after();
      if (mine) x.scores_gradient(tP, ctl->stats[2 * s + h][1] + u * kCols, m);
      else store_zeros(tP);
      hand_over(b.bar(kDSDone));
    }
    if (ok) {
      ok = __all_sync(0xffffffffu, ptx::mbar_wait(b.bar(kFinal), 0, b.abort_flag));
      if (!ok && lane == 0) report(a.status, 7, 2 + h, -1);
    }
    if (!ok) return;
    ptx::tc_fence_after();
    const int grow = b.row0 + wq * 32 + lane;
    const int64_t at = (static_cast<int64_t>(b.bh) * a.N + grow) * D * 2;
    const int col = (2 * h + u) * 32;
    auto to = [&](void* g) { return reinterpret_cast<uint4*>(static_cast<unsigned char*>(g) + at + 2 * col); };
    const uint32_t t = b.tmem + lane_base + col;
    store_rows<kBF16, 32>(t + 256, b.count > 0, grow < a.N, a.scale, to(a.dk));
    store_rows<kBF16, 32>(t + 384, b.count > 0, grow < a.N, kBF16 ? 1.f : exp2f(-kHalfShift), to(a.dv));
  }
};

template <int D, bool kBF16>
__global__ void __launch_bounds__(kThreads<D>, 1) sparse_attn_bwd_kernel(
    const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
    const __grid_constant__ CUtensorMap tm_do, const __grid_constant__ BwdArgs a) {
  using Queries = Chains<D, kBF16, false>;
  extern __shared__ unsigned char smem_raw[];
  Block b;
  b.smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Control* ctl = reinterpret_cast<Control*>(b.smem + kTilesBytes<D>);
  b.bar0 = ptx::smem_u32(&ctl->bars[0]);
  b.abort_flag = &ctl->abort_flag;

  const int warp = ptx::warp_index();
  const int lane = threadIdx.x % 32;
  const Item it = item_of(a);
  const Lists& l = it.keys ? a.key_lists : a.query_lists;
  const int nlist = it.keys ? a.ntiles : (a.ntiles + 1) / 2;
  const int index = it.keys ? it.pos : it.pos >> 1;
  const int item = l.order ? __ldg(l.order + index) : index;
  const int mh = item / nlist;
  const int tile = it.keys ? item - mh * nlist : 2 * (item - mh * nlist) + (it.pos & 1);
  if (tile >= a.ntiles) return;                   // the second query tile of a pair that has one only
  const int kv_max = max(a.kvl_lo, a.kvl_hi);
  b.bh = it.batch * a.Hm + mh;
  b.row0 = tile * kTile;
  b.blocks = ctl->blocks;

  auto with_kind = [&](auto&& f) {
    if (it.keys) {
      if constexpr (D == 128) f(Pairs<kBF16>{});
      else f(Chains<64, kBF16, true>{});
    } else {
      f(Queries{});
    }
  };
  if (threadIdx.x == 0) {
    with_kind([&](auto kind) {
      for (int i = 0; i < kNumBarriers; ++i) ptx::mbar_init(b.bar(i), kind.arrivals(i));
    });
    ctl->abort_flag = 0;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&tm_q);
    ptx::prefetch_tensormap(&tm_k);
    ptx::prefetch_tensormap(&tm_v);
    ptx::prefetch_tensormap(&tm_do);
  }
  if (warp == 2) {
    ptx::tmem_alloc(ptx::smem_u32(&ctl->tmem_base), 512);
    ptx::tmem_relinquish();
    ptx::tc_fence_before();
  }
  Fixed<D> fixed;
  if (warp >= 4 && !it.keys) fixed.load(a, b.bh, b.row0);
  if (warp == 3) {
    const int32_t* ent = l.entries + static_cast<int64_t>(item) * a.ntiles;
    int n = it.keys ? expand<true>(ent, l.counts + item, a.ntiles, 0, a.N, ctl->blocks)
                          : expand<false>(ent, l.counts + item, a.ntiles, 4 * (it.pos & 1), kv_max, ctl->blocks);
    n = (it.keys && b.row0 >= kv_max) ? 0 : n;    // keys that no row may see
    if ((a.kvl_lo + kBlock - 1) / kBlock != (a.kvl_hi + kBlock - 1) / kBlock) n = visible(a, it.keys, b.row0, n, ctl->blocks);
    if (lane == 0) ctl->count = n;
  }
  __syncthreads();
  ptx::tc_fence_after();
  asm volatile("griddepcontrol.wait;" ::: "memory");      // for the row statistics: nothing above may read them
  b.tmem = ctl->tmem_base;
  b.count = ctl->count;

  if (warp == 0) {
    if (ptx::elect_one()) {
      with_kind([&](auto kind) {
        if (it.keys) kind.produce(b, a, ctl, &tm_k, &tm_v, &tm_q, &tm_do);
        else kind.produce(b, a, ctl, nullptr, nullptr, &tm_k, &tm_v);
      });
    }
  } else if (warp == 1) {
    if (ptx::elect_one()) with_kind([&](auto kind) { kind.issue(b, a, 0); });
  } else if (warp == 3) {
    if (ptx::elect_one()) with_kind([&](auto kind) { kind.issue(b, a, 1); });
  } else if (warp >= 4) {
    with_kind([&](auto kind) { kind.compute(b, a, ctl, fixed, warp, lane); });
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(b.tmem, 512);
  }
}

// Row statistics: one group of D / 8 threads per row.  Rows past N and rows that attend to nothing get -inf, so that their
// probabilities are zero whatever the scores are.
template <int D, bool kBF16>
__global__ void __launch_bounds__(256) bwd_stats_kernel(const void* __restrict__ out, const void* __restrict__ lo,
                                                        const void* __restrict__ dout, const float* __restrict__ lse, int N, int npad,
                                                        float* __restrict__ nlse, float* __restrict__ ndelta) {
  asm volatile("griddepcontrol.launch_dependents;");      // the items may set themselves up meanwhile
  constexpr int kTpr = D / 8;
  const int bh = blockIdx.y;
  const int row = blockIdx.x * (256 / kTpr) + threadIdx.x / kTpr;
  const int c = threadIdx.x % kTpr;
  float sum = 0.f;
  if (row < N) {
    const int64_t at = (static_cast<int64_t>(bh) * N + row) * kTpr + c;
    const uint4 a = __ldg(static_cast<const uint4*>(out) + at), b = __ldg(static_cast<const uint4*>(dout) + at);
    const uint4 r = lo ? __ldg(static_cast<const uint4*>(lo) + at) : make_uint4(0, 0, 0, 0);
    const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w}, wr[4] = {r.x, r.y, r.z, r.w};
    auto floats = [](const uint32_t& w) {
      if constexpr (kBF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
      else return __half22float2(*reinterpret_cast<const __half2*>(&w));
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = floats(wa[i]), y = floats(wb[i]), z = floats(wr[i]);
      sum = fmaf(x.x + z.x, y.x, sum);
      sum = fmaf(x.y + z.y, y.y, sum);
    }
  }
#pragma unroll
  for (int o = kTpr / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (c == 0 && row < npad) {
    const int64_t to = static_cast<int64_t>(bh) * npad + row;
    const float l = row < N ? lse[static_cast<int64_t>(bh) * N + row] : -INFINITY;
    const bool empty = l == -INFINITY;
    nlse[to] = empty ? -INFINITY : (kBF16 ? 0.f : kHalfShift) - l * kLog2e;
    ndelta[to] = empty ? 0.f : (kBF16 ? -sum : -sum * exp2f(-kHalfShift));
  }
}

template <int D, bool kBF16>
int launch(BwdArgs a, const void* out, const void* lo, const float* lse, int dtype, int BH, float* ws, cudaStream_t st) {
  const int kv_rows = max(1, max(a.kvl_lo, a.kvl_hi));
  CUtensorMap tq, tk, tv, tdo;
  if (int rc = make_tmap_rows(&tq, a.q, dtype, BH, a.N, D, kBlock)) return rc;
  if (int rc = make_tmap_rows(&tdo, a.dout, dtype, BH, a.N, D, kBlock)) return rc;
  if (int rc = make_tmap_first_rows(&tk, a.k, dtype, BH, a.N, kv_rows, D, kBlock)) return rc;
  if (int rc = make_tmap_first_rows(&tv, a.v, dtype, BH, a.N, kv_rows, D, kBlock)) return rc;
  auto kernel = sparse_attn_bwd_kernel<D, kBF16>;
  const size_t smem = kTilesBytes<D> + 1024 + sizeof(Control);
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return rc;
  a.nlse = ws;
  a.ndelta = ws + static_cast<int64_t>(BH) * a.npad;
  bwd_stats_kernel<D, kBF16><<<dim3(a.npad / (2048 / D), BH), 256, 0, st>>>(out, lo, a.dout, lse, a.N, a.npad, ws,
                                                                                  ws + static_cast<int64_t>(BH) * a.npad);
  MODDIT_CHECK_LAUNCH("bwd_stats_kernel");
  const int64_t blocks = static_cast<int64_t>(2 * a.ntiles + (a.ntiles & 1)) * BH;
  // Launched beside the statistics: barriers, tensor memory and block lists are ready when these are.  2 heads of 4,096 at D = 128
  // 58.8 -> 57.6 us, 1,200 rows 23.3 -> 22.7; the next launch of the stream still waits for all of it.
  cudaLaunchAttribute beside{};
  beside.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  beside.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(blocks));
  config.blockDim = dim3(kThreads<D>);
  config.dynamicSmemBytes = smem;
  config.stream = st;
  config.attrs = &beside;
  config.numAttrs = 1;
  (void)cudaLaunchKernelEx(&config, kernel, tq, tk, tv, tdo, a);
  MODDIT_CHECK_LAUNCH("sparse_attn_bwd_kernel");
  return MODDIT_OK;
}

}  // namespace
}  // namespace moddit

using namespace moddit;

extern "C" size_t moddit_sparse_attn_bwd_workspace_bytes(int BH, int N) {
  if (BH <= 0 || N <= 0) return 0;
  return static_cast<size_t>(2) * BH * ceil_div(N, kTile) * kTile * sizeof(float);
}

extern "C" int moddit_sparse_attn_bwd(const void* q, const void* k, const void* v, const void* out, const void* out_lo,
                                      const void* dout, const float* lse, int dtype, int BH, int N, int D, const int32_t* q_counts,
                                      const int32_t* q_entries, const int32_t* q_order, const int32_t* k_counts,
                                      const int32_t* k_entries, const int32_t* k_order, int Hm, float softmax_scale,
                                      int q_split, int kv_len_lo, int kv_len_hi, void* dq, void* dk, void* dv, void* workspace,
                                      size_t workspace_bytes, int32_t* status, void* stream) {
  clear_error();
  MODDIT_CHECK_ARG(q && k && v && out && dout && lse && q_counts && q_entries && k_counts && k_entries && dq && dk && dv && status,
                   "sparse_attn_bwd: null pointer");
  MODDIT_CHECK_ARG(BH > 0 && BH <= 65535 && N > 0 && Hm > 0, "sparse_attn_bwd: BH=%d N=%d Hm=%d out of range", BH, N, Hm);
  MODDIT_CHECK_ARG(BH % Hm == 0, "sparse_attn_bwd: BH=%d is not a multiple of the mask heads Hm=%d", BH, Hm);
  MODDIT_CHECK_ARG(softmax_scale > 0.f, "sparse_attn_bwd: softmax_scale must be positive");
  MODDIT_CHECK_ARG(kv_len_lo >= 0 && kv_len_lo <= N && kv_len_hi >= 0 && kv_len_hi <= N,
                   "sparse_attn_bwd: kv_len (%d, %d) outside [0, N=%d]", kv_len_lo, kv_len_hi, N);
  if (D != 64 && D != 128) return fail(MODDIT_E_UNSUPPORTED, "sparse_attn_bwd: head_dim must be 64 or 128, got %d", D);
  if (dtype != MODDIT_BF16 && dtype != MODDIT_FP16) return fail(MODDIT_E_ARG, "sparse_attn_bwd: unknown dtype %d", dtype);
  static_assert(kMaxBlocks * kBlock == MODDIT_ATTN_BWD_MAX_ROWS, "rows of a work item's block list");
  if (N > MODDIT_ATTN_BWD_MAX_ROWS)
    return fail(MODDIT_E_UNSUPPORTED, "sparse_attn_bwd: N=%d exceeds %d", N, MODDIT_ATTN_BWD_MAX_ROWS);
  if (static_cast<int64_t>(2 * ceil_div(N, kTile) + 1) * BH > (1ll << 31) - 1)
    return fail(MODDIT_E_UNSUPPORTED, "sparse_attn_bwd: %d heads of %d rows are too many work items", BH, N);
  const void* tensors[9] = {q, k, v, out, out_lo, dout, dq, dk, dv};
  for (const void* p : tensors)
    if (!aligned16(p)) return fail(MODDIT_E_ALIGN, "sparse_attn_bwd: all (BH, N, D) tensors must be 16-byte aligned");
  if (workspace == nullptr || workspace_bytes < moddit_sparse_attn_bwd_workspace_bytes(BH, N) || !aligned16(workspace))
    return fail(MODDIT_E_WORKSPACE, "sparse_attn_bwd: a 16-byte aligned workspace of %zu bytes is needed",
                moddit_sparse_attn_bwd_workspace_bytes(BH, N));
  if (int rc = require_sm100()) return rc;
  BwdArgs a{};
  a.key_lists = Lists{k_counts, k_entries, k_order};
  a.query_lists = Lists{q_counts, q_entries, q_order};
  a.q = q; a.k = k; a.v = v; a.dout = dout;
  a.dq = dq; a.dk = dk; a.dv = dv; a.status = status;
  a.Hm = Hm; a.batches = BH / Hm; a.N = N;
  a.ntiles = ceil_div(N, kTile); a.npad = a.ntiles * kTile;
  a.q_split = q_split; a.kvl_lo = kv_len_lo; a.kvl_hi = kv_len_hi;
  a.scale = softmax_scale; a.scale_log2 = softmax_scale * kLog2e;
  float* ws = static_cast<float*>(workspace);
  cudaStream_t st = as_stream(stream);
  if (D == 128)
    return dtype == MODDIT_BF16 ? launch<128, true>(a, out, out_lo, lse, dtype, BH, ws, st) : launch<128, false>(a, out, out_lo, lse, dtype, BH, ws, st);
  return dtype == MODDIT_BF16 ? launch<64, true>(a, out, out_lo, lse, dtype, BH, ws, st) : launch<64, false>(a, out, out_lo, lse, dtype, BH, ws, st);
}
