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
// into memory with atomics (at 2,560 clocks of tensor pipe a tile about 25 bytes a clock and SM, and sums whose order varies).
//
// Both kinds share one program: a block holds two fixed tiles (F0, F1 = K, V or Q, dO) and streams pairs of tiles
// (X0, X1 = Q, dO or K, V):   S = F0 X0^T,  dP = F1 X1^T,  acc1 += P X1 (key items),  acc0 += dS X0.
// P and dS stay in tensor memory, 16 bits wide, over the scores they came from, as the A operand of the second products;
// X0 and X1 serve as K-major operands of the first products and as MN-major operands of the second from one copy in shared
// memory.
// Roles (12 warps): 0 TMA producer, 1 MMA issuer, 2 tensor-memory allocation, 4-11 elementwise: thread = row (lane) and 64 of
// the tile's 128 columns.
// Tensor memory (512 columns): S [0,128) dP [128,256) acc0 [256,256+D) acc1 [384,384+D); P and dS overwrite columns
// [64 h, 64 h + 32) of S and dP for column half h.
// The issue order  acc1 += P(e) X1, S(e+1), acc0 += dS(e) X0, dP(e+1)  keeps the tensor pipe busy with the first two while
// dS(e) is computed and with the other two while P(e+1) is.
//
// Sums are float32 in tensor memory; P and dS are rounded to the inputs' type once, for the second products.  P <= 1 falls
// with the number of keys: for float16 it is held 2^8 times larger (its normal range then reaches 2^-22) and the factor is
// taken out of dS before its rounding and of dV at the end.
// Every wait is bounded (ptx::mbar_wait) and reports as in the forward.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace moddit {
namespace {

constexpr int kThreads = 384;
constexpr int kTile = 128;
constexpr int kStages = 2;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHalfShift = 8.f;      // float16: P is held 2^kHalfShift times larger

enum BarrierIndex {
  kFixed = 0,                         // F0, F1 have landed
  kFull,                              // [kStages] X0, X1 (and the row statistics of a key item) have landed
  kEmpty = kFull + kStages,           // [kStages] all products of an entry are done
  kSFull = kEmpty + kStages,          // scores are ready
  kDPFull,                            // dP is ready
  kPDone,                             // S has been read and P stored
  kDSDone,                            // dP has been read and dS stored
  kFinal,
  kNumBarriers
};

struct __align__(16) Control {
  float stats[kStages][2][kTile];     // key items: -lse * log2 e and -delta of the streamed query rows
  unsigned long long bars[kNumBarriers];
  uint32_t tmem_base;
  int abort_flag;
};

template <int D>
constexpr size_t smem_bytes() {
  return static_cast<size_t>(2 + 2 * kStages) * kTile * D * 2 + 1024 + sizeof(Control);
}

struct BwdArgs {
  const int32_t* counts;
  const int32_t* entries;
  const int32_t* order;
  const float* nlse;                  // (BH, npad): -lse * log2 e (+ kHalfShift), -inf for rows that attend to nothing
  const float* ndelta;                // (BH, npad): -delta (* 2^-kHalfShift)
  void* g0;                           // dK or dQ
  void* g1;                           // dV
  int32_t* status;
  int Hm, N, ntiles, npad, q_split, kvl_lo, kvl_hi;
  float scale, scale_log2;
};

__device__ __forceinline__ void report(int32_t* status, int code, int role, int where) {
  if (atomicCAS(status, 0, code) == 0) {
    status[1] = static_cast<int32_t>(blockIdx.y * gridDim.x + blockIdx.x);
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

// Row statistics: one group of D / 8 threads per row.  Rows past N and rows that attend to nothing get -inf, so that their
// probabilities are zero whatever the scores are.
template <int D, bool kBF16>
__global__ void __launch_bounds__(256) bwd_stats_kernel(const void* __restrict__ out, const void* __restrict__ dout,
                                                        const float* __restrict__ lse, int N, int npad,
                                                        float* __restrict__ nlse, float* __restrict__ ndelta) {
  constexpr int kTpr = D / 8;
  const int bh = blockIdx.y;
  const int row = blockIdx.x * (256 / kTpr) + threadIdx.x / kTpr;
  const int c = threadIdx.x % kTpr;
  float sum = 0.f;
  if (row < N) {
    const int64_t at = (static_cast<int64_t>(bh) * N + row) * kTpr + c;
    const uint4 a = __ldg(static_cast<const uint4*>(out) + at), b = __ldg(static_cast<const uint4*>(dout) + at);
    const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 x, y;
      if constexpr (kBF16) {
        x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&wa[i]));
        y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&wb[i]));
      } else {
        x = __half22float2(*reinterpret_cast<const __half2*>(&wa[i]));
        y = __half22float2(*reinterpret_cast<const __half2*>(&wb[i]));
      }
      sum = fmaf(x.x, y.x, sum);
      sum = fmaf(x.y, y.y, sum);
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

template <int D, bool kBF16, bool kKeys>
__global__ void __launch_bounds__(kThreads, 1) sparse_attn_bwd_kernel(
    const __grid_constant__ CUtensorMap tm_f0, const __grid_constant__ CUtensorMap tm_f1,
    const __grid_constant__ CUtensorMap tm_x0, const __grid_constant__ CUtensorMap tm_x1,
    const __grid_constant__ BwdArgs a) {
  constexpr int kTileBytes = kTile * D * 2;
  constexpr int kChunks = D / 64;                 // 64-element (128-byte) column chunks per tile
  constexpr int kChunkBytes = kTile * 128;
  constexpr uint32_t kIdescS = ptx::idesc_f16(128, 128, kBF16, false);
  constexpr uint32_t kIdescG = ptx::idesc_f16(128, D, kBF16, true);

  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Control* ctl = reinterpret_cast<Control*>(smem + (2 + 2 * kStages) * kTileBytes);
  const uint32_t sF = ptx::smem_u32(smem);
  const uint32_t sX = sF + 2 * kTileBytes;        // stage s: X0 at sX + 2 s tiles, X1 behind it
  const uint32_t bar0 = ptx::smem_u32(&ctl->bars[0]);
  auto bar = [&](int i) { return bar0 + 8u * static_cast<uint32_t>(i); };
  volatile int* abort_flag = &ctl->abort_flag;

  const int warp = ptx::warp_index();
  const int lane = threadIdx.x % 32;
  // work item: key items are listed by tile, query items by pair of tiles
  const int nlist = kKeys ? a.ntiles : (a.ntiles + 1) / 2;
  const int index = kKeys ? blockIdx.x : blockIdx.x >> 1;
  const int item = a.order ? a.order[index] : index;
  const int mh = item / nlist;
  const int tile = kKeys ? item - mh * nlist : 2 * (item - mh * nlist) + (blockIdx.x & 1);
  const int fshift = kKeys ? 0 : 4 * (blockIdx.x & 1);
  if (tile >= a.ntiles) return;
  const int bh = blockIdx.y * a.Hm + mh;
  const int row0 = tile * kTile;
  int cnt = a.counts[item];
  if (kKeys && row0 >= max(a.kvl_lo, a.kvl_hi)) cnt = 0;
  const int32_t* ent = a.entries + static_cast<int64_t>(item) * a.ntiles;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kNumBarriers; ++i) ptx::mbar_init(bar(i), (i == kPDone || i == kDSDone) ? 256u : 1u);
    ctl->abort_flag = 0;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&tm_f0);
    ptx::prefetch_tensormap(&tm_f1);
    ptx::prefetch_tensormap(&tm_x0);
    ptx::prefetch_tensormap(&tm_x1);
  }
  if (warp == 2) {
    ptx::tmem_alloc(ptx::smem_u32(&ctl->tmem_base), 512);
    ptx::tmem_relinquish();
    ptx::tc_fence_before();
  }
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = ctl->tmem_base;
  auto flags_of = [&](int en) { return (en >> fshift) & 0xf; };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (ptx::elect_one() && cnt > 0) {
      ptx::mbar_expect_tx(bar(kFixed), 2 * kTileBytes);
      for (int c = 0; c < kChunks; ++c) {
        ptx::tma_load_3d(sF + c * kChunkBytes, &tm_f0, bar(kFixed), c * 64, row0, bh);
        ptx::tma_load_3d(sF + kTileBytes + c * kChunkBytes, &tm_f1, bar(kFixed), c * 64, row0, bh);
      }
      bool ok = true;
      int n = 0;
      for (int e = 0; e < cnt && ok; ++e) {
        if (!flags_of(ent[e])) continue;
        const int s = n % kStages;
        ok = ptx::mbar_wait(bar(kEmpty + s), ((n / kStages) & 1) ^ 1, abort_flag);
        if (!ok) { report(a.status, 1, 0, e); break; }
        const int x0 = (ent[e] >> 8) * kTile;
        const uint32_t to = sX + 2 * s * kTileBytes;
        ptx::mbar_expect_tx(bar(kFull + s), 2 * kTileBytes + (kKeys ? 2 * kTile * 4 : 0));
        for (int c = 0; c < kChunks; ++c) {
          ptx::tma_load_3d(to + c * kChunkBytes, &tm_x0, bar(kFull + s), c * 64, x0, bh);
          ptx::tma_load_3d(to + kTileBytes + c * kChunkBytes, &tm_x1, bar(kFull + s), c * 64, x0, bh);
        }
        if (kKeys) {
          const int64_t at = static_cast<int64_t>(bh) * a.npad + x0;
          ptx::bulk_load(ptx::smem_u32(ctl->stats[s][0]), a.nlse + at, kTile * 4, bar(kFull + s));
          ptx::bulk_load(ptx::smem_u32(ctl->stats[s][1]), a.ndelta + at, kTile * 4, bar(kFull + s));
        }
        ++n;
      }
      if (!ok) {
        // give copies in flight a bounded time to land (their barriers may never be consumed)
        for (int i = 0; i < 4096 && !ptx::mbar_try_wait(bar(kFixed), 0); ++i) {}
        for (int m = max(0, n - kStages); m < n; ++m)
          for (int i = 0; i < 4096 && !ptx::mbar_try_wait(bar(kFull + m % kStages), (m / kStages) & 1); ++i) {}
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (ptx::elect_one()) {
      auto advance = [](uint64_t desc, uint32_t bytes) -> uint64_t {
        return (desc & 0xffffffff00000000ull) | static_cast<uint32_t>(static_cast<uint32_t>(desc) + (bytes >> 4));
      };
      const uint64_t df = ptx::smem_desc_sw128(sF, 16, 1024);              // K-major: F0, F1 and the X tiles
      const uint64_t dx = advance(df, sX - sF);
      const uint64_t dg = ptx::smem_desc_sw128(sX, kChunkBytes, 1024);     // MN-major: the X tiles
      // which = 0: S = F0 X0^T, 1: dP = F1 X1^T
      auto first = [&](int which, int s) {
        const uint64_t a0 = advance(df, which * kTileBytes), b0 = advance(dx, (2 * s + which) * kTileBytes);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk / 4) * kChunkBytes + (kk % 4) * 32;
          ptx::mma_ss(tmem + which * 128, advance(a0, off), advance(b0, off), kIdescS, kk > 0 ? 1u : 0u);
        }
        ptx::tc_commit(bar(kSFull + which));
      };
      // which = 0: acc1 += P X1, 1: acc0 += dS X0
      auto second = [&](int which, int s, uint32_t acc) {
        const uint64_t b0 = advance(dg, (2 * s + 1 - which) * kTileBytes);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          ptx::mma_ts(tmem + (which ? 256 : 384), tmem + which * 128 + (kk / 4) * 64 + (kk % 4) * 8, advance(b0, kk * 2048),
                      kIdescG, (acc || kk > 0) ? 1u : 0u);
      };
      bool ok = true;
      int e = 0, n = 0;
      auto next_kept = [&](int from) {
        while (from < cnt && !flags_of(ent[from])) ++from;
        return from;
      };
      e = next_kept(0);
      if (e < cnt) {
        ok = ptx::mbar_wait(bar(kFixed), 0, abort_flag) && ptx::mbar_wait(bar(kFull), 0, abort_flag);
        if (!ok) report(a.status, 2, 1, -1);
        ptx::tc_fence_after();
        if (ok) { first(0, 0); first(1, 0); }
      }
      while (e < cnt && ok) {
        const int s = n % kStages, s1 = (n + 1) % kStages;
        const int e1 = next_kept(e + 1);
        const bool next = e1 < cnt;
        ok = ptx::mbar_wait(bar(kPDone), n & 1, abort_flag);
        if (!ok) { report(a.status, 3, 1, e); break; }
        ptx::tc_fence_after();
        if (kKeys) second(0, s, n > 0);
        if (next) {
          ok = ptx::mbar_wait(bar(kFull + s1), ((n + 1) / kStages) & 1, abort_flag);
          if (!ok) { report(a.status, 2, 1, e); break; }
          ptx::tc_fence_after();
          first(0, s1);
        }
        ok = ptx::mbar_wait(bar(kDSDone), n & 1, abort_flag);
        if (!ok) { report(a.status, 3, 1, e); break; }
        ptx::tc_fence_after();
        second(1, s, n > 0);
        ptx::tc_commit(bar(kEmpty + s));
        if (next) first(1, s1);
        e = e1;
        ++n;
      }
      ptx::tc_commit(bar(kFinal));
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ elementwise
    const int h = (warp - 4) / 4;                 // column half
    const int r = (warp % 4) * 32 + lane;         // row inside the tile
    const int grow = row0 + r;
    const uint32_t lane_base = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t tS = tmem + lane_base + h * 64;
    const uint32_t tP = tS + 128;
    const int kv_min = min(a.kvl_lo, a.kvl_hi);
    // bit of the sub-block that this thread's row and columns lie in
    const int keep_bit = kKeys ? 2 * h + (r >> 6) : 2 * (r >> 6) + h;
    float nl_row = 0.f, nd_row = 0.f;
    if (!kKeys) {
      nl_row = a.nlse[static_cast<int64_t>(bh) * a.npad + grow];
      nd_row = a.ndelta[static_cast<int64_t>(bh) * a.npad + grow];
    }
    const uint64_t scale2 = ptx::pack_f32x2(a.scale_log2, a.scale_log2);
    const uint64_t nl2 = ptx::pack_f32x2(nl_row, nl_row), nd2 = ptx::pack_f32x2(nd_row, nd_row);
    const float kDown = kBF16 ? 1.f : 1.f / 256.f;
    const uint64_t down2 = ptx::pack_f32x2(kDown, kDown);
    bool ok = true;
    int n = 0;
    for (int e = 0; e < cnt; ++e) {
      const int fl = flags_of(ent[e]);
      if (!fl) continue;
      const int s = n % kStages;
      const int x0 = (ent[e] >> 8) * kTile;
      // columns [0, keep_below) and [keep_from, 64) of this thread are kept
      int keep_below = 64, keep_from = 64;
      if (fl != 0xf || (kKeys ? row0 : x0) + kTile > kv_min) {
        if (!((fl >> keep_bit) & 1)) {
          keep_below = 0;
        } else if (kKeys) {
          const int split = min(max(a.q_split - x0 - 64 * h, 0), 64);
          keep_below = grow < a.kvl_lo ? split : 0;
          keep_from = grow < a.kvl_hi ? split : 64;
        } else {
          keep_below = (grow < a.q_split ? a.kvl_lo : a.kvl_hi) - x0 - 64 * h;
        }
      }
      const bool whole = keep_below >= keep_from || keep_below >= 64;
      const bool any_masked = __any_sync(0xffffffffu, !whole);
      if (kKeys) ok = ptx::mbar_wait(bar(kFull + s), (n / kStages) & 1, abort_flag);      // the statistics
      ok = ok && ptx::mbar_wait(bar(kSFull), n & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) { if (lane == 0) report(a.status, 4, 2 + h, e); break; }
      ptx::tc_fence_after();
      float p[64];
#pragma unroll
      for (int c = 0; c < 2; ++c) ptx::tmem_ld32(tS + c * 32, reinterpret_cast<uint32_t*>(p) + c * 32);
      ptx::tmem_ld_wait();
      const ulonglong2* nlv = reinterpret_cast<const ulonglong2*>(ctl->stats[s][0] + 64 * h);
      const ulonglong2* ndv = reinterpret_cast<const ulonglong2*>(ctl->stats[s][1] + 64 * h);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const ulonglong2 nl = kKeys ? nlv[i] : make_ulonglong2(nl2, nl2);
        float x0f, x1f, x2f, x3f;
        ptx::unpack_f32x2(ptx::fma_f32x2(ptx::pack_f32x2(p[4 * i], p[4 * i + 1]), scale2, nl.x), x0f, x1f);
        ptx::unpack_f32x2(ptx::fma_f32x2(ptx::pack_f32x2(p[4 * i + 2], p[4 * i + 3]), scale2, nl.y), x2f, x3f);
        p[4 * i] = ptx::ex2(x0f);
        p[4 * i + 1] = ptx::ex2(x1f);
        p[4 * i + 2] = ptx::ex2(x2f);
        p[4 * i + 3] = ptx::ex2(x3f);
      }
      if (any_masked) {
#pragma unroll
        for (int c = 0; c < 64; ++c) p[c] = (c < keep_below || c >= keep_from) ? p[c] : 0.f;
      }
      if (kKeys) {
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) pk[i] = pack2<kBF16>(p[2 * i], p[2 * i + 1]);
        ptx::tmem_st32(tS, pk);
        ptx::tmem_st_wait();
      }
      ptx::tc_fence_before();
      ptx::mbar_arrive(bar(kPDone));

      ok = ptx::mbar_wait(bar(kDPFull), n & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) { if (lane == 0) report(a.status, 5, 2 + h, e); break; }
      ptx::tc_fence_after();
      float d[64];
#pragma unroll
      for (int c = 0; c < 2; ++c) ptx::tmem_ld32(tP + c * 32, reinterpret_cast<uint32_t*>(d) + c * 32);
      ptx::tmem_ld_wait();
      if (any_masked) {                           // what lies in a masked place may be anything
#pragma unroll
        for (int c = 0; c < 64; ++c) d[c] = (c < keep_below || c >= keep_from) ? d[c] : 0.f;
      }
      uint32_t dk[32];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const ulonglong2 nd = kKeys ? ndv[i] : make_ulonglong2(nd2, nd2);
        uint64_t t0 = ptx::pack_f32x2(d[4 * i], d[4 * i + 1]), t1 = ptx::pack_f32x2(d[4 * i + 2], d[4 * i + 3]);
        t0 = kBF16 ? ptx::add_f32x2(t0, nd.x) : ptx::fma_f32x2(t0, down2, nd.x);
        t1 = kBF16 ? ptx::add_f32x2(t1, nd.y) : ptx::fma_f32x2(t1, down2, nd.y);
        t0 = ptx::mul_f32x2(t0, ptx::pack_f32x2(p[4 * i], p[4 * i + 1]));
        t1 = ptx::mul_f32x2(t1, ptx::pack_f32x2(p[4 * i + 2], p[4 * i + 3]));
        float y0, y1, y2, y3;
        ptx::unpack_f32x2(t0, y0, y1);
        ptx::unpack_f32x2(t1, y2, y3);
        dk[2 * i] = pack2<kBF16>(y0, y1);
        dk[2 * i + 1] = pack2<kBF16>(y2, y3);
      }
      ptx::tmem_st32(tP, dk);
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      ptx::mbar_arrive(bar(kDSDone));
      ++n;
    }
    if (ok) {
      ok = ptx::mbar_wait(bar(kFinal), 0, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok && lane == 0) report(a.status, 6, 2 + h, -1);
    }
    if (ok) {
      ptx::tc_fence_after();
      const float g1_scale = kBF16 ? 1.f : exp2f(-kHalfShift);
      // accumulator `which` of D columns: half h of the warps stores half of them
#pragma unroll
      for (int which = 0; which < (kKeys ? 2 : 1); ++which) {
        const float f = which ? g1_scale : a.scale;
        uint4* dst = reinterpret_cast<uint4*>(static_cast<unsigned char*>(which ? a.g1 : a.g0) +
                                              (static_cast<int64_t>(bh) * a.N + grow) * D * 2) + h * (D / 16);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          float o[32];
          if (n > 0) {
            ptx::tmem_ld32(tmem + lane_base + (which ? 384 : 256) + h * (D / 2) + c * 32, reinterpret_cast<uint32_t*>(o));
            ptx::tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.f;
          }
          if (grow < a.N) {
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
              uint4 w;
              w.x = pack2<kBF16>(o[q4 * 8 + 0] * f, o[q4 * 8 + 1] * f);
              w.y = pack2<kBF16>(o[q4 * 8 + 2] * f, o[q4 * 8 + 3] * f);
              w.z = pack2<kBF16>(o[q4 * 8 + 4] * f, o[q4 * 8 + 5] * f);
              w.w = pack2<kBF16>(o[q4 * 8 + 6] * f, o[q4 * 8 + 7] * f);
              dst[c * 4 + q4] = w;
            }
          }
        }
      }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

struct Lists {
  const int32_t *counts, *entries, *order;
};

template <int D, bool kBF16>
int launch(const void* q, const void* k, const void* v, const void* out, const void* dout, const float* lse, int dtype, int BH,
           int N, const Lists& ql, const Lists& kl, int Hm, float softmax_scale, int q_split, int kvl_lo, int kvl_hi, void* dq,
           void* dk, void* dv, float* ws, int32_t* status, cudaStream_t st) {
  const int nt = ceil_div(N, kTile), npad = nt * kTile;
  const int kv_rows = max(1, max(kvl_lo, kvl_hi));
  CUtensorMap tq, tk, tv, tdo;
  if (int rc = make_tmap_rows(&tq, q, dtype, BH, N, D, kTile)) return rc;
  if (int rc = make_tmap_rows(&tdo, dout, dtype, BH, N, D, kTile)) return rc;
  if (int rc = make_tmap_first_rows(&tk, k, dtype, BH, N, kv_rows, D, kTile)) return rc;
  if (int rc = make_tmap_first_rows(&tv, v, dtype, BH, N, kv_rows, D, kTile)) return rc;
  float* nlse = ws;
  float* ndelta = ws + static_cast<int64_t>(BH) * npad;
  bwd_stats_kernel<D, kBF16><<<dim3(npad / (2048 / D), BH), 256, 0, st>>>(out, dout, lse, N, npad, nlse, ndelta);
  MODDIT_CHECK_LAUNCH("bwd_stats_kernel");
  BwdArgs a{};
  a.nlse = nlse; a.ndelta = ndelta; a.status = status;
  a.Hm = Hm; a.N = N; a.ntiles = nt; a.npad = npad; a.q_split = q_split; a.kvl_lo = kvl_lo; a.kvl_hi = kvl_hi;
  a.scale = softmax_scale; a.scale_log2 = softmax_scale * kLog2e;
  const size_t smem = smem_bytes<D>();
  auto keys = sparse_attn_bwd_kernel<D, kBF16, true>;
  auto queries = sparse_attn_bwd_kernel<D, kBF16, false>;
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(keys), smem)) return rc;
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(queries), smem)) return rc;
  a.counts = kl.counts; a.entries = kl.entries; a.order = kl.order; a.g0 = dk; a.g1 = dv;
  keys<<<dim3(nt * Hm, BH / Hm), kThreads, smem, st>>>(tk, tv, tq, tdo, a);
  MODDIT_CHECK_LAUNCH("sparse_attn_bwd_kernel (keys)");
  a.counts = ql.counts; a.entries = ql.entries; a.order = ql.order; a.g0 = dq; a.g1 = nullptr;
  queries<<<dim3(2 * ((nt + 1) / 2) * Hm, BH / Hm), kThreads, smem, st>>>(tq, tdo, tk, tv, a);
  MODDIT_CHECK_LAUNCH("sparse_attn_bwd_kernel (queries)");
  return MODDIT_OK;
}

}  // namespace
}  // namespace moddit

using namespace moddit;

extern "C" size_t moddit_sparse_attn_bwd_workspace_bytes(int BH, int N) {
  if (BH <= 0 || N <= 0) return 0;
  return static_cast<size_t>(2) * BH * ceil_div(N, kTile) * kTile * sizeof(float);
}

extern "C" int moddit_sparse_attn_bwd(const void* q, const void* k, const void* v, const void* out, const void* dout,
                                      const float* lse, int dtype, int BH, int N, int D, const int32_t* q_counts,
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
  const void* tensors[8] = {q, k, v, out, dout, dq, dk, dv};
  for (const void* p : tensors)
    if (!aligned16(p)) return fail(MODDIT_E_ALIGN, "sparse_attn_bwd: all (BH, N, D) tensors must be 16-byte aligned");
  if (workspace == nullptr || workspace_bytes < moddit_sparse_attn_bwd_workspace_bytes(BH, N) || !aligned16(workspace))
    return fail(MODDIT_E_WORKSPACE, "sparse_attn_bwd: a 16-byte aligned workspace of %zu bytes is needed",
                moddit_sparse_attn_bwd_workspace_bytes(BH, N));
  if (int rc = require_sm100()) return rc;
  const Lists ql{q_counts, q_entries, q_order}, kl{k_counts, k_entries, k_order};
  float* ws = static_cast<float*>(workspace);
  cudaStream_t st = as_stream(stream);
#define MODDIT_BWD(DIM, BF16)                                                                                             \
  launch<DIM, BF16>(q, k, v, out, dout, lse, dtype, BH, N, ql, kl, Hm, softmax_scale, q_split, kv_len_lo, kv_len_hi, dq, dk, \
                    dv, ws, status, st)
  if (D == 128) return dtype == MODDIT_BF16 ? MODDIT_BWD(128, true) : MODDIT_BWD(128, false);
  return dtype == MODDIT_BF16 ? MODDIT_BWD(64, true) : MODDIT_BWD(64, false);
#undef MODDIT_BWD
}
