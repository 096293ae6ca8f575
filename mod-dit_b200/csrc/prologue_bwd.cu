// Gradients of the attention prologue (prologue.cu): the rotary embedding turned back, the normalisation's gradient, the
// move from the head-major to the token-major layout and the gradients of the norm's weight and bias, in one pass over the
// data.  With g the gradient of a row after the rotation is turned back, x the projection, w the weight, r the row's factor:
//   rms    r = rsqrt(mean(x^2) + eps)          dx = r g w - x r^3 mean(g w x)
//   layer  xhat = (x - mean) r                 dx = r (g w - mean(g w) - xhat mean(g w xhat))
//   dw = sum over rows of g xhat (xhat = x r for rms),   db = sum of g
// The forward's intermediate roundings to the 16-bit type count as the identity; the factors are computed again in float32
// from x, so the forward keeps nothing for this pass but its inputs.
//
// Bound: HBM.  Algorithmic bytes per token: q and k 3 * 2 * H * D each (g and x in, dx out), v 2 * 2 * H * D; the rotary
// tables are fetched once for all heads.  57,728 tokens of 16 x 128 (one fused projection, rms per head) 320 - 327 us = 6.0 - 6.1
// TB/s, 91 - 93 % of the measured copy bandwidth; 2 x 45,104 of 30 x 64 (layer) 466 - 524 us = 5.3 - 6.0 TB/s; without a norm
// 57,728 tokens of 16 x 128 242 us = 6.1 TB/s.
//
// Weight gradients are sums over all tokens.  Blocks are persistent: a thread keeps float32 sums for the eight columns it
// always has, a block adds its threads' sums in shared memory and writes one row of partial sums, and a second kernel adds
// the rows in index order: the results are the same bits on every run.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"

namespace moddit {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 2;                // rows per thread of an item of the per-head kernel
constexpr int kStages = 5;              // heads of them in flight
constexpr int kWide = 640;              // threads of the kernel with a piece of a whole token each

template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 floats(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ __nv_bfloat16 round(float a) { return __float2bfloat16_rn(a); }
};
template <>
struct Pair<__half> {
  static __device__ __forceinline__ float2 floats(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ __half round(float a) { return __float2half_rn(a); }
};

template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = Pair<T>::floats(w[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(Pair<T>::pack(f[0], f[1]), Pair<T>::pack(f[2], f[3]), Pair<T>::pack(f[4], f[5]), Pair<T>::pack(f[6], f[7]));
}

// Sum over an aligned group of kLanes lanes of a warp.
template <int kLanes>
__device__ __forceinline__ float lane_sum(float x) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

struct BwdArgs {
  const void* g[3];        // (B, H, N_out, D)
  const void* x[2];        // token-major, token_stride elements between tokens; null without a norm
  void* dx[3];             // token-major, out_stride elements between tokens
  const void* weight[2];
  float* part[2];          // partial sums: gridDim.x rows of dw, then as many of db
  const float* cos;
  const float* sin;
  int64_t token_stride, out_stride;
  int B, S, H, N_out, src_row0, rope_form, rope_lo, rope_hi;
  int heads_per_item;      // of the per-head kernel
  float eps;
};

// The factors that turn a pair's gradients back, for columns 8 c to 8 c + 7 of token s: the forward has
//   out0 = y0 cs0 - y1 sn0,  out1 = y0 sn1 + y1 cs1,  so  dy0 = g0 cs0 + g1 sn1,  dy1 = g1 cs1 - g0 sn0.
struct Turn {
  float cs[8], sn[8];
};
// kPair: tables of one value per pair (MODDIT_ROPE_PAIR)
template <int D, bool kPair>
__device__ __forceinline__ Turn turn_of(const BwdArgs& a, int s, int c) {
  Turn t;
  if (a.cos == nullptr || s < a.rope_lo || s >= a.rope_hi) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t.cs[i] = 1.f, t.sn[i] = 0.f;
    return t;
  }
  if constexpr (kPair) {
    const int64_t at = static_cast<int64_t>(s - a.rope_lo) * (D / 2) + c * 4;
    const float4 c4 = __ldg(reinterpret_cast<const float4*>(a.cos + at)), s4 = __ldg(reinterpret_cast<const float4*>(a.sin + at));
    const float cv[4] = {c4.x, c4.y, c4.z, c4.w}, sv[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t.cs[2 * i] = t.cs[2 * i + 1] = cv[i];
      t.sn[2 * i] = t.sn[2 * i + 1] = sv[i];
    }
  } else {
    const int64_t at = static_cast<int64_t>(s - a.rope_lo) * D + c * 8;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      *reinterpret_cast<float4*>(t.cs + i) = __ldg(reinterpret_cast<const float4*>(a.cos + at + i));
      *reinterpret_cast<float4*>(t.sn + i) = __ldg(reinterpret_cast<const float4*>(a.sin + at + i));
    }
    if (a.rope_form == MODDIT_ROPE_EVEN_COS_ODD_SIN) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        t.cs[2 * i + 1] = t.cs[2 * i];
        t.sn[2 * i] = t.sn[2 * i + 1];
      }
    }
  }
  return t;
}
__device__ __forceinline__ uint4 load16(const void* p, bool in) {
  return in ? __ldg(static_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ void turn_back(const Turn& t, float (&g)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float g0 = g[2 * i], g1 = g[2 * i + 1];
    g[2 * i] = g0 * t.cs[2 * i] + g1 * t.sn[2 * i + 1];
    g[2 * i + 1] = g1 * t.cs[2 * i + 1] - g0 * t.sn[2 * i];
  }
}

// 16 bytes into shared memory, zeros where `in` is false (src is not read then)
__device__ __forceinline__ void copy_async16(void* dst, const void* src, bool in) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(__cvta_generic_to_global(src)), "r"(in ? 16 : 0)
               : "memory");
}

// Grid: x = persistent blocks, y = tensor.  An item is kRows rows per thread of `heads_per_item` heads: a thread has the same
// columns of the same tokens in every head, so the rotary factors are read once and stay in registers (float32 tables of D
// values weigh more per row and head than the rows themselves: through the L2 for every head they were the bound).  A thread
// copies its pieces of the next kStages - 1 heads asynchronously into places of its own in shared memory, so that bytes are in
// flight while it computes, without registers for them and without a barrier.  57,728 tokens x 16 heads of 128: loads into
// registers, two heads at a time, 400 us; like this 320.
template <typename T, int D, int kNorm, bool kPair>
__global__ void __launch_bounds__(kThreads, 2) prologue_bwd_kernel(const __grid_constant__ BwdArgs a) {
  constexpr int kTpr = D / 8;                     // threads per row
  constexpr int kRpp = kThreads / kTpr;           // rows per pass
  constexpr float kInvD = 1.0f / D;
  extern __shared__ uint4 ring[];                 // [kStages][kRows][g, x][kThreads]; at the end the sums of kRpp rows
  const int which = blockIdx.y;
  const T* __restrict__ g_in = static_cast<const T*>(a.g[which]);
  if (g_in == nullptr) return;
  T* __restrict__ dx = static_cast<T*>(a.dx[which]);
  const int c = threadIdx.x % kTpr, rg = threadIdx.x / kTpr;
  const bool normed = kNorm != MODDIT_NORM_NONE && which < 2;
  const bool turned = which < 2 && a.cos != nullptr;
  const T* __restrict__ x_in = normed ? static_cast<const T*>(a.x[which]) : nullptr;
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (normed && a.weight[which] != nullptr) unpack<T>(__ldg(static_cast<const uint4*>(a.weight[which]) + c), w);
  float dw[8] = {}, db[8] = {};

  auto work = [&](uint4 gv, uint4 xv, const Turn& turn, bool in) -> uint4 {
    float g[8];
    unpack<T>(gv, g);
    if (turned) turn_back(turn, g);
    if (normed) {
      float x[8];
      unpack<T>(xv, x);
      if constexpr (kNorm == MODDIT_NORM_RMS_HEAD) {
        float ss = 0.f, sg = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss = fmaf(x[i], x[i], ss);
          sg = fmaf(g[i] * w[i], x[i], sg);
        }
        const float ms = lane_sum<kTpr>(ss) * kInvD;
        const float r = in ? rsqrtf(ms + a.eps) : 0.f;     // rows past the end add nothing, eps = 0 included
        const float f = -r * r * (lane_sum<kTpr>(sg) * kInvD);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dw[i] = fmaf(g[i], x[i] * r, dw[i]);
          g[i] = r * fmaf(x[i], f, g[i] * w[i]);
        }
      } else if constexpr (kNorm == MODDIT_NORM_LAYER) {
        float sx = 0.f, sg = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sx += x[i];
          sg = fmaf(g[i], w[i], sg);
        }
        const float mean = lane_sum<kTpr>(sx) * kInvD, mg = lane_sum<kTpr>(sg) * kInvD;
        float ss = 0.f, sgx = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] -= mean;
          ss = fmaf(x[i], x[i], ss);
          sgx = fmaf(g[i] * w[i], x[i], sgx);
        }
        const float ms = lane_sum<kTpr>(ss) * kInvD;
        const float r = in ? rsqrtf(ms + a.eps) : 0.f;
        const float f = -r * r * (lane_sum<kTpr>(sgx) * kInvD);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dw[i] = fmaf(g[i], x[i] * r, dw[i]);
          db[i] += g[i];
          g[i] = r * (fmaf(x[i], f, g[i] * w[i]) - mg);
        }
      }
    }
    return pack8<T>(g);
  };

  const int tiles = (a.S + kRows * kRpp - 1) / (kRows * kRpp);
  const int chunks = (a.H + a.heads_per_item - 1) / a.heads_per_item;
  const int64_t items = static_cast<int64_t>(a.B) * tiles * chunks;
  const int64_t head_rows = static_cast<int64_t>(a.N_out) * D;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int chunk = static_cast<int>(item % chunks);
    const int64_t bt = item / chunks;
    const int b = static_cast<int>(bt / tiles);
    const int s0 = static_cast<int>(bt - static_cast<int64_t>(b) * tiles) * kRows * kRpp + rg;
    const int h0 = chunk * a.heads_per_item, h1 = min(a.H, h0 + a.heads_per_item);
    const T *gp[kRows], *xp[kRows];
    T* dp[kRows];
    bool in[kRows];
    Turn turn[kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int s = s0 + u * kRpp;
      const int64_t tok = static_cast<int64_t>(b) * a.S + s;
      in[u] = s < a.S;
      gp[u] = g_in + (static_cast<int64_t>(b) * a.H * a.N_out + a.src_row0 + s) * D + c * 8;
      xp[u] = x_in + tok * a.token_stride + c * 8;
      dp[u] = dx + tok * a.out_stride + c * 8;
      if (turned) turn[u] = turn_of<D, kPair>(a, s, c);
    }
    auto fetch = [&](int h) {
      if (h < h1) {
        uint4* to = ring + ((h - h0) % kStages) * (2 * kRows * kThreads) + threadIdx.x;
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          copy_async16(to + 2 * u * kThreads, in[u] ? gp[u] + h * head_rows : g_in, in[u]);
          if (normed) copy_async16(to + (2 * u + 1) * kThreads, in[u] ? xp[u] + h * D : x_in, in[u]);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int j = 0; j < kStages - 1; ++j) fetch(h0 + j);
    for (int h = h0; h < h1; ++h) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      const uint4* from = ring + ((h - h0) % kStages) * (2 * kRows * kThreads) + threadIdx.x;
      uint4 gv[kRows], xv[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        gv[u] = from[2 * u * kThreads];
        if (normed) xv[u] = from[(2 * u + 1) * kThreads];
      }
      fetch(h + kStages - 1);
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const uint4 res = (normed || turned) ? work(gv[u], xv[u], turn[u], in[u]) : gv[u];
        if (in[u]) *reinterpret_cast<uint4*>(dp[u] + h * D) = res;
      }
    }
  }
  if (normed && a.part[which] != nullptr) {
    float* red = reinterpret_cast<float*>(ring);
    for (int k = 0; k < (kNorm == MODDIT_NORM_LAYER ? 2 : 1); ++k) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) red[rg * D + c * 8 + i] = k ? db[i] : dw[i];
      __syncthreads();
      if (threadIdx.x < D) {
        float t = 0.f;
        for (int j = 0; j < kRpp; ++j) t += red[j * D + threadIdx.x];
        a.part[which][(static_cast<int64_t>(k) * gridDim.x + blockIdx.x) * D + threadIdx.x] = t;
      }
    }
  }
}

// Normalisation over all heads of a token.  A block has one token per warp at a time.  First every warp sums x^2 and g w x
// over its token; then a thread takes fixed pieces of eight columns through the block's tokens, whose rows it reads again
// (from the L2), writes dx and adds to its columns' weight gradient, which lives in shared memory.  A piece lies at the same
// columns of its head for all pieces of a lane or thread, so the rotary factors are read once a token: in the second part from
// shared memory, where the first part's lanes have put them.
// For tokens too wide for the kernel below.  8,192 tokens of 48 x 128 186 us, 67 % of the measured copy bandwidth; 4,096 of
// 64 x 128 141 us, 58 %; 4,096 of 128 x 128 279 us, 59 %; bound by instructions and the two parts' latencies.  At 8,640 of 40 x
// 128, which the kernel below has now, it took 172 us.
// Slower: a group's rows kept in shared memory between the parts, copied a group ahead (204 us with two blocks an SM, 257 with
// one: block-wide sums and fewer warps), half as many tokens in flight with three or four blocks an SM (190 - 230).
template <typename T, int D, bool kPair>
__global__ void __launch_bounds__(kThreads, 2) prologue_bwd_all_heads_kernel(const __grid_constant__ BwdArgs a) {
  constexpr int kTpr = D / 8;
  constexpr int kTokens = kThreads / 32;
  constexpr int kBatch = 4;                       // pieces in flight per lane in the first part
  extern __shared__ float dw_s[];                 // H * D
  __shared__ float r_s[kTokens], f_s[kTokens];
  __shared__ __align__(16) float cs_s[kTokens][D], sn_s[kTokens][D];
  const int which = blockIdx.y;
  const T* __restrict__ g_in = static_cast<const T*>(a.g[which]);
  if (g_in == nullptr) return;
  const T* __restrict__ x_in = which < 2 ? static_cast<const T*>(a.x[which]) : nullptr;
  T* __restrict__ dx = static_cast<T*>(a.dx[which]);
  const uint4* wp = which < 2 ? static_cast<const uint4*>(a.weight[which]) : nullptr;
  const int W = a.H * D, pieces = W / 8;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const bool sums = which < 2 && a.part[which] != nullptr;
  const bool turned = which < 2 && a.cos != nullptr;
  if (sums)
    for (int i = threadIdx.x; i < W; i += kThreads) dw_s[i] = 0.f;
  const float inv_w = 1.f / static_cast<float>(W);
  const int groups = (a.S + kTokens - 1) / kTokens;
  const int64_t head_rows = static_cast<int64_t>(a.N_out) * D;
  auto weights = [&](int p, float (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.f;
    if (wp != nullptr) unpack<T>(__ldg(wp + p), w);
  };
  for (int64_t grp = blockIdx.x; grp < static_cast<int64_t>(a.B) * groups; grp += gridDim.x) {
    const int b = static_cast<int>(grp / groups);
    const int s0 = static_cast<int>(grp - static_cast<int64_t>(b) * groups) * kTokens;
    const T* g0 = g_in + (static_cast<int64_t>(b) * a.H * a.N_out + a.src_row0 + s0) * D;        // token s0 of head 0
    const T* x0 = x_in + (static_cast<int64_t>(b) * a.S + s0) * a.token_stride;
    T* d0 = dx + (static_cast<int64_t>(b) * a.S + s0) * a.out_stride;
    if (which < 2) {
      const bool in = s0 + warp < a.S;
      const Turn turn = turn_of<D, kPair>(a, in ? s0 + warp : -1, lane % kTpr);
      float ss = 0.f, sg = 0.f;
      const T* gp = g0 + (lane / kTpr) * head_rows + warp * D + (lane % kTpr) * 8;
      const T* xp = x0 + warp * a.token_stride + lane * 8;
      const int64_t step = (32 / kTpr) * head_rows;
      for (int p0 = lane; p0 < pieces && in; p0 += 32 * kBatch) {
        uint4 gv[kBatch], xv[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const bool there = p0 + 32 * j < pieces;
          gv[j] = load16(gp, there);
          xv[j] = load16(xp + j * 256, there);
          gp += step;
        }
        xp += kBatch * 256;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          float g[8], x[8], w[8];
          unpack<T>(gv[j], g);
          unpack<T>(xv[j], x);
          weights(min(p0 + 32 * j, pieces - 1), w);
          if (turned) turn_back(turn, g);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            ss = fmaf(x[i], x[i], ss);
            sg = fmaf(g[i] * w[i], x[i], sg);
          }
        }
      }
      ss = lane_sum<32>(ss);
      sg = lane_sum<32>(sg);
      __syncthreads();                            // the previous group's factors have been read
      if (turned && lane < kTpr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          cs_s[warp][lane * 8 + i] = turn.cs[i];
          sn_s[warp][lane * 8 + i] = turn.sn[i];
        }
      }
      if (lane == 0) {
        const float r = in ? rsqrtf(ss * inv_w + a.eps) : 0.f;
        r_s[warp] = r;
        f_s[warp] = -r * r * (sg * inv_w);
      }
      __syncthreads();
    }
    for (int p = threadIdx.x; p < pieces; p += kThreads) {
      const int c = p % kTpr;
      const T* gp = g0 + (p / kTpr) * head_rows + c * 8;
      uint4 gv[kTokens], xv[kTokens];
#pragma unroll
      for (int t = 0; t < kTokens; ++t) {
        const bool in = s0 + t < a.S;
        gv[t] = load16(gp + t * D, in);
        if (which < 2) xv[t] = load16(x0 + t * a.token_stride + p * 8, in);
      }
      float w[8], dw[8] = {};
      if (which < 2) weights(p, w);
#pragma unroll
      for (int t = 0; t < kTokens; ++t) {
        uint4 res = gv[t];
        if (which < 2) {
          float g[8], x[8];
          unpack<T>(gv[t], g);
          unpack<T>(xv[t], x);
          if (turned) {
            Turn turn;
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
              *reinterpret_cast<float4*>(turn.cs + i) = *reinterpret_cast<const float4*>(&cs_s[t][c * 8 + i]);
              *reinterpret_cast<float4*>(turn.sn + i) = *reinterpret_cast<const float4*>(&sn_s[t][c * 8 + i]);
            }
            turn_back(turn, g);
          }
          const float r = r_s[t], f = f_s[t];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float xr = x[i] * r;
            dw[i] = fmaf(g[i], xr, dw[i]);
            g[i] = fmaf(xr, f, r * (g[i] * w[i]));
          }
          res = pack8<T>(g);
        }
        if (s0 + t < a.S) *reinterpret_cast<uint4*>(d0 + t * a.out_stride + p * 8) = res;
      }
      if (sums)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw_s[p * 8 + i] += dw[i];
    }
  }
  if (sums) {
    __syncthreads();
    for (int i = threadIdx.x; i < W; i += kThreads) a.part[which][static_cast<int64_t>(blockIdx.x) * W + i] = dw_s[i];
  }
}

// The same for tokens of up to kWide pieces, in one pass over the rows: a thread has one piece of eight columns of every token of
// its block, kept from the sums to dx in registers, with its columns' weights and weight gradient.  Two tokens at a time share
// one block-wide sum of four values and one barrier.  The rows of the next kStages - 1 pairs of tokens are on their way into
// places of the thread's own in shared memory, as in the per-head kernel, and with them the two tokens' rows of the rotary
// tables, once a block.  Where q, k and v are all given, a block of q or k also copies one token of v per pair of its own:
// copies want bytes, the sums want instructions.
// 8,640 tokens of 40 x 128: 129 - 139 us, 5.1 - 5.5 TB/s, 78 - 84 % of the measured copy bandwidth; 260 instructions a piece, issued in 0.65 of
// the cycles, are the other bound.  On the way: divisions and products for every pair's addresses, rotary rows loaded per thread
// 170 us; those loaded a pair ahead 158 (spills where a table has a value a column); pointers moved on by additions 154; rotary
// rows through shared memory 145; v beside q and k 137; q and k at once, half of the blocks each, 130.  Slower: two operations
// an instruction on packed pairs (more registers: spills, 194 us against 158).
template <typename T, int D, bool kPair>
__global__ void __launch_bounds__(kWide, 1) prologue_bwd_tokens_kernel(const __grid_constant__ BwdArgs a) {
  constexpr int kTpr = D / 8;
  constexpr int kRow = kPair ? D / 2 : D;         // floats of a row of the rotary tables
  constexpr int kChunks = 4 * kRow / 4;           // pieces of 16 bytes of two tokens' rows of both
  extern __shared__ uint4 ring[];                 // [kStages][2][g, x][threads], then [kStages][2][cos, sin][kRow] floats
  __shared__ float red[2][4][kWide / 32];         // [round & 1][x^2, g w x of the first token, of the second][warp]
  const int which = blockIdx.y, threads = blockDim.x;
  const T* __restrict__ g_in = static_cast<const T*>(a.g[which]);
  const bool beside = a.g[0] && a.g[1] && a.g[2];   // the blocks of q and k copy a token of v each along with a pair of theirs
  if (g_in == nullptr || (beside && which == 2)) return;
  const bool normed = which < 2, turned = which < 2 && a.cos != nullptr;
  const T* __restrict__ x_in = normed ? static_cast<const T*>(a.x[which]) : nullptr;
  T* __restrict__ dx = static_cast<T*>(a.dx[which]);
  const int W = a.H * D;
  const bool has = threadIdx.x < W / 8;
  const int p = has ? threadIdx.x : 0, c = p % kTpr;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = threads / 32;
  const float inv_w = 1.f / static_cast<float>(W);
  float w[8], dw[8] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (normed && has && a.weight[which] != nullptr) unpack<T>(__ldg(static_cast<const uint4*>(a.weight[which]) + p), w);

  // A block has every gridDim.x-th pair of tokens.  The pointers to where it reads (`ahead`) and writes (`at`) are moved on by
  // additions, and made anew where the sample changes.
  const int even = (a.S + 1) / 2 * 2, step = 2 * gridDim.x;
  struct Place {
    int b, s;
    __device__ bool next(int step, int S) {       // true where the sample has changed
      s += step;
      if (s < S) return false;
      do s -= S, ++b;
      while (s >= S);
      return true;
    }
  };
  Place at{0, 0};
  at.next(2 * blockIdx.x, even);
  Place ahead = at;
  const int64_t head = static_cast<int64_t>(p / kTpr) * a.N_out + a.src_row0;
  const int64_t x_step = step * a.token_stride, d_step = step * a.out_stride;
  auto g_at = [&](const Place& of) { return g_in + (static_cast<int64_t>(of.b) * a.H * a.N_out + head + of.s) * D + c * 8; };
  auto x_at = [&](const Place& of) { return x_in + (static_cast<int64_t>(of.b) * a.S + of.s) * a.token_stride + p * 8; };
  auto d_at = [&](const Place& of) { return dx + (static_cast<int64_t>(of.b) * a.S + of.s) * a.out_stride + p * 8; };
  const T *gp = g_at(ahead), *xp = x_at(ahead);
  T* dp = d_at(at);
  const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(ring + threadIdx.x)), apart = 16 * threads;
  auto copy = [&](uint32_t to, const void* from, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(__cvta_generic_to_global(from)), "r"(in ? 16 : 0)
                 : "memory");
  };
  const uint4* const tables = ring + kStages * 4 * threads;
  const uint32_t tables_at = static_cast<uint32_t>(__cvta_generic_to_shared(tables));
  auto turned_at = [&](int s) { return turned && s >= a.rope_lo && s < a.rope_hi; };
  auto fetch = [&](int stage) {
    if (ahead.b < a.B) {
      if (turned)
        for (int i = threadIdx.x; i < kChunks; i += threads) {
          const int s = ahead.s + i / (kChunks / 2), piece = i % (kRow / 4);
          const float* from = i / (kRow / 4) % 2 ? a.sin : a.cos;
          const bool in = turned_at(s);
          copy(tables_at + 16 * (stage * kChunks + i), in ? from + static_cast<int64_t>(s - a.rope_lo) * kRow + 4 * piece : from, in);
        }
      const uint32_t to = mine + stage * 4 * apart;
      const bool two = ahead.s + 1 < a.S;
      copy(to, gp, has);
      copy(to + 2 * apart, two ? gp + D : gp, two && has);
      if (normed) {
        copy(to + apart, xp, has);
        copy(to + 3 * apart, two ? xp + a.token_stride : xp, two && has);
      }
      if (ahead.next(step, even)) {
        gp = g_at(ahead);
        xp = x_at(ahead);
      } else {
        gp += step * D;
        xp += x_step;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int j = 0; j < kStages - 1; ++j) fetch(j);
  int stage = 0, round = 0;
  auto turn_at = [&](int stage, int t) {
    const float4* row = reinterpret_cast<const float4*>(tables + stage * kChunks + t * (kChunks / 2));
    Turn f;
    if constexpr (kPair) {
      const float4 cs = row[c], sn = row[kRow / 4 + c];
      const float cv[4] = {cs.x, cs.y, cs.z, cs.w}, sv[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f.cs[2 * i] = f.cs[2 * i + 1] = cv[i];
        f.sn[2 * i] = f.sn[2 * i + 1] = sv[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        *reinterpret_cast<float4*>(f.cs + 4 * i) = row[2 * c + i];
        *reinterpret_cast<float4*>(f.sn + 4 * i) = row[kRow / 4 + 2 * c + i];
      }
      if (a.rope_form == MODDIT_ROPE_EVEN_COS_ODD_SIN) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f.cs[2 * i + 1] = f.cs[2 * i];
          f.sn[2 * i] = f.sn[2 * i + 1];
        }
      }
    }
    return f;
  };
  // The tables' rows are copied by one thread and read by others: a round waits for the next round's copies before its barrier.
  asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
  __syncthreads();
  for (; at.b < a.B; round ^= 1) {
    const int s0 = at.s;
    T* const to = dp;
    const bool copies = beside && has && s0 + which < a.S;
    uint4 copied;
    int64_t vrow = 0;
    if (copies) {
      copied = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.g[2]) + (static_cast<int64_t>(at.b) * a.H * a.N_out + head + s0 + which) * D + c * 8));
      vrow = static_cast<int64_t>(at.b) * a.S + s0 + which;
    }
    if (at.next(step, even)) dp = d_at(at);
    else dp += d_step;
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 3) : "memory");
    const uint4* from = ring + stage * 4 * threads + threadIdx.x;
    uint4 gv[2], xv[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      gv[t] = from[2 * t * threads];
      if (normed) xv[t] = from[(2 * t + 1) * threads];
    }
    const int now = stage;
    fetch(stage == 0 ? kStages - 1 : stage - 1);
    stage = stage == kStages - 1 ? 0 : stage + 1;
    if (normed) {
      float g[2][8], sum[4] = {};
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float x[8];
        unpack<T>(gv[t], g[t]);
        unpack<T>(xv[t], x);
        if (turned_at(s0 + t)) turn_back(turn_at(now, t), g[t]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sum[2 * t] = fmaf(x[i], x[i], sum[2 * t]);
          sum[2 * t + 1] = fmaf(g[t][i] * w[i], x[i], sum[2 * t + 1]);
        }
      }
      // four sums over the warp in six exchanges: eight lanes end with each of them
      const bool up = lane & 16, odd = lane & 8;
      const float s = (up ? sum[2] : sum[0]) + __shfl_xor_sync(0xffffffffu, up ? sum[0] : sum[2], 16);
      const float d = (up ? sum[3] : sum[1]) + __shfl_xor_sync(0xffffffffu, up ? sum[1] : sum[3], 16);
      const float part = lane_sum<8>((odd ? d : s) + __shfl_xor_sync(0xffffffffu, odd ? s : d, 8));
      if (lane % 8 == 0) red[round][lane / 8][warp] = part;
      __syncthreads();
      float all = 0.f;
      for (int j = lane % 8; j < warps; j += 8) all += red[round][lane / 8][j];
      all = lane_sum<8>(all);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float ss = __shfl_sync(0xffffffffu, all, 16 * t), sg = __shfl_sync(0xffffffffu, all, 16 * t + 8);
        const float r = s0 + t < a.S ? rsqrtf(ss * inv_w + a.eps) : 0.f;     // a token past the end adds nothing, eps = 0 included
        const float f = -r * r * (sg * inv_w);
        float x[8];
        unpack<T>(xv[t], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float xr = x[i] * r;
          dw[i] = fmaf(g[t][i], xr, dw[i]);
          g[t][i] = fmaf(xr, f, r * (g[t][i] * w[i]));
        }
        gv[t] = pack8<T>(g[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
      if (has && s0 + t < a.S) *reinterpret_cast<uint4*>(to + t * a.out_stride) = gv[t];
    if (copies) *reinterpret_cast<uint4*>(static_cast<T*>(a.dx[2]) + vrow * a.out_stride + p * 8) = copied;
  }
  if (normed && has && a.part[which] != nullptr) {
    float4* to = reinterpret_cast<float4*>(a.part[which] + static_cast<int64_t>(blockIdx.x) * W + p * 8);
    to[0] = make_float4(dw[0], dw[1], dw[2], dw[3]);
    to[1] = make_float4(dw[4], dw[5], dw[6], dw[7]);
  }
}

// Adds the rows of partial sums in index order: 32 columns a block, eight groups of rows.  y = tensor, z = weight, bias.
struct SumArgs {
  const float* part[2];
  void* out[2][2];
};
template <typename T>
__global__ void __launch_bounds__(kThreads) prologue_bwd_sums_kernel(const __grid_constant__ SumArgs a, int rows, int width) {
  __shared__ float red[8][32];
  T* out = static_cast<T*>(a.out[blockIdx.y][blockIdx.z]);
  if (out == nullptr) return;
  const int col = blockIdx.x * 32 + threadIdx.x % 32, grp = threadIdx.x / 32;
  const float* p = a.part[blockIdx.y] + static_cast<int64_t>(blockIdx.z) * rows * width;
  float t = 0.f;
#pragma unroll 8
  for (int j = grp; j < rows; j += 8) t += p[static_cast<int64_t>(j) * width + col];
  red[grp][threadIdx.x % 32] = t;
  __syncthreads();
  if (grp == 0) {
#pragma unroll
    for (int j = 1; j < 8; ++j) t += red[j][threadIdx.x];
    out[col] = Pair<T>::round(t);
  }
}

// Persistent blocks per tensor: a fixed number, whatever the GPU, so that the order of the sums does not depend on it; more
// than the items of a tensor would only add rows of zeros.  Short inputs are cut into fewer heads per item, so that there are
// that many.
constexpr int kBlocksPerHead = 296;
constexpr int kBlocksAllHeads = 296;
constexpr int kBlocksTokens = 148;                   // q's and k's half of them each where both are given
constexpr int kMaxWidth = MODDIT_TOKEN_NORM_BWD_MAX_WIDTH;       // values of a token: their sums lie in shared memory
int heads_per_item(int B, int S, int H, int D) {
  const int64_t tiles = static_cast<int64_t>(B) * ceil_div(S, kRows * kThreads / (D / 8));
  const int chunks = static_cast<int>(std::min<int64_t>(H, (kBlocksPerHead + tiles - 1) / tiles));
  return ceil_div(H, chunks);
}
// Tokens of up to kWide pieces are read once (a thread a piece), wider ones twice.  8,640 tokens of 40 x 128: 130 us once, 172
// twice; 32,760 of 12 x 128: 148 and 235; 40,000 of 16 x 64: 128 and 233; 1,000 of 12 x 128 alike.
bool one_pass(int H, int D) { return H <= kWide * 8 / D; }
int token_threads(int H, int D) { return ceil_div(H * D / 8, 32) * 32; }
constexpr size_t token_smem(int threads, int floats) { return sizeof(uint4) * kStages * (4 * threads + floats); }
// as many blocks an SM as its registers and 227 KB of shared memory hold
int token_blocks(int threads) {
  return std::max(1, std::min(kWide / threads, static_cast<int>(226 * 1024 / (token_smem(threads, 128) + 2048))));
}
int blocks_for(int B, int S, int H, int D, int norm_kind, int tensors = 1) {
  if (norm_kind == MODDIT_NORM_RMS_ALL_HEADS && one_pass(H, D))
    return static_cast<int>(std::min<int64_t>(kBlocksTokens * token_blocks(token_threads(H, D)) / tensors,
                                              static_cast<int64_t>(B) * ceil_div(S, 2)));
  if (norm_kind == MODDIT_NORM_RMS_ALL_HEADS)
    return static_cast<int>(std::min<int64_t>(kBlocksAllHeads, static_cast<int64_t>(B) * ceil_div(S, kThreads / 32)));
  return static_cast<int>(std::min<int64_t>(kBlocksPerHead, static_cast<int64_t>(B) * ceil_div(S, kRows * kThreads / (D / 8)) *
                                                                ceil_div(H, heads_per_item(B, S, H, D))));
}

template <typename T, int D, bool kPair>
int launch_rows(const BwdArgs& a, int norm_kind, int blocks, cudaStream_t st) {
  if (norm_kind == MODDIT_NORM_RMS_ALL_HEADS && one_pass(a.H, D)) {
    auto kernel = prologue_bwd_tokens_kernel<T, D, kPair>;
    const int threads = token_threads(a.H, D);
    const size_t smem = token_smem(threads, a.cos == nullptr ? 0 : kPair ? D / 2 : D);
    if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return rc;
    kernel<<<dim3(blocks, 3), threads, smem, st>>>(a);
  } else if (norm_kind == MODDIT_NORM_RMS_ALL_HEADS) {
    auto kernel = prologue_bwd_all_heads_kernel<T, D, kPair>;
    const size_t smem = sizeof(float) * a.H * D;
    if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return rc;
    kernel<<<dim3(blocks, 3), kThreads, smem, st>>>(a);
  } else {
    auto kernel = norm_kind == MODDIT_NORM_NONE       ? prologue_bwd_kernel<T, D, MODDIT_NORM_NONE, kPair>
                  : norm_kind == MODDIT_NORM_RMS_HEAD ? prologue_bwd_kernel<T, D, MODDIT_NORM_RMS_HEAD, kPair>
                                                      : prologue_bwd_kernel<T, D, MODDIT_NORM_LAYER, kPair>;
    const size_t smem = sizeof(uint4) * kStages * kRows * 2 * kThreads;
    if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return rc;
    kernel<<<dim3(blocks, 3), kThreads, smem, st>>>(a);
  }
  return MODDIT_OK;
}

template <typename T, int D>
int launch_bwd(const BwdArgs& a, int norm_kind, int blocks, const SumArgs& sums, cudaStream_t st) {
  const bool pair = a.rope_form == MODDIT_ROPE_PAIR;
  if (int rc = pair ? launch_rows<T, D, true>(a, norm_kind, blocks, st) : launch_rows<T, D, false>(a, norm_kind, blocks, st)) return rc;
  MODDIT_CHECK_LAUNCH("prologue_bwd_kernel");
  if (sums.out[0][0] || sums.out[0][1] || sums.out[1][0] || sums.out[1][1]) {
    const int width = norm_kind == MODDIT_NORM_RMS_ALL_HEADS ? a.H * D : D;
    prologue_bwd_sums_kernel<T><<<dim3(width / 32, 2, norm_kind == MODDIT_NORM_LAYER ? 2 : 1), kThreads, 0, st>>>(sums, blocks, width);
    MODDIT_CHECK_LAUNCH("prologue_bwd_sums_kernel");
  }
  return MODDIT_OK;
}

}  // namespace
}  // namespace moddit

using namespace moddit;

extern "C" size_t moddit_qkv_prologue_bwd_workspace_bytes(int B, int S, int H, int D, int norm_kind) {
  if (B <= 0 || S <= 0 || H <= 0 || (D != 64 && D != 128) || norm_kind <= MODDIT_NORM_NONE || norm_kind > MODDIT_NORM_LAYER) return 0;
  const size_t width = norm_kind == MODDIT_NORM_RMS_ALL_HEADS ? static_cast<size_t>(H) * D : 2 * D;
  return 2 * width * blocks_for(B, S, H, D, norm_kind) * sizeof(float);
}

extern "C" int moddit_qkv_prologue_bwd(const void* dq, const void* dk, const void* dv, const void* q_in, const void* k_in,
                                       int dtype, int B, int S, int H, int D, int64_t token_stride, int norm_kind,
                                       const void* q_weight, const void* k_weight, float eps, const float* rope_cos,
                                       const float* rope_sin, int rope_form, int rope_lo, int rope_hi, int N_out, int src_row0,
                                       void* dq_in, void* dk_in, void* dv_in, int64_t out_stride, void* dq_weight,
                                       void* dq_bias, void* dk_weight, void* dk_bias, void* workspace, size_t ws_bytes,
                                       void* stream) {
  clear_error();
  MODDIT_CHECK_ARG(dtype == MODDIT_BF16 || dtype == MODDIT_FP16, "dtype must be MODDIT_BF16 or MODDIT_FP16");
  MODDIT_CHECK_ARG(D == 64 || D == 128, "head_dim %d not supported (64 or 128)", D);
  MODDIT_CHECK_ARG(B > 0 && S > 0 && H > 0, "B, S and H must be positive (got %d, %d, %d)", B, S, H);
  MODDIT_CHECK_ARG(norm_kind >= MODDIT_NORM_NONE && norm_kind <= MODDIT_NORM_LAYER, "unknown norm_kind %d", norm_kind);
  MODDIT_CHECK_ARG(dq != nullptr || dk != nullptr || dv != nullptr, "no gradient given");
  MODDIT_CHECK_ARG(src_row0 >= 0 && static_cast<int64_t>(src_row0) + S <= N_out, "rows %d..%lld are not in tensors of %d rows",
                   src_row0, static_cast<long long>(src_row0) + S, N_out);
  const int64_t width = static_cast<int64_t>(H) * D;
  MODDIT_CHECK_ARG(out_stride >= width && out_stride % 8 == 0, "out_stride %lld must be a multiple of 8 elements and at least H*D",
                   static_cast<long long>(out_stride));
  const void* g[3] = {dq, dk, dv};
  const void* x[2] = {q_in, k_in};
  void* dx[3] = {dq_in, dk_in, dv_in};
  for (int i = 0; i < 3; ++i) {
    if (g[i] == nullptr) continue;
    MODDIT_CHECK_ARG(dx[i] != nullptr, "gradient %d has no output buffer", i);
    MODDIT_CHECK_ARG(aligned16(g[i]) && aligned16(dx[i]), "tensor %d is not 16-byte aligned", i);
    if (i < 2 && norm_kind != MODDIT_NORM_NONE) {
      MODDIT_CHECK_ARG(x[i] != nullptr && aligned16(x[i]), "input %d of the normalisation is null or not 16-byte aligned", i);
      MODDIT_CHECK_ARG(token_stride >= width && token_stride % 8 == 0,
                       "token_stride %lld must be a multiple of 8 elements and at least H*D", static_cast<long long>(token_stride));
    }
  }
  MODDIT_CHECK_ARG(aligned16(q_weight) && aligned16(k_weight), "norm parameters must be 16-byte aligned");
  void* grads[2][2] = {{dq_weight, dq_bias}, {dk_weight, dk_bias}};
  bool any = false;
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j) {
      if (grads[i][j] == nullptr) continue;
      any = true;
      MODDIT_CHECK_ARG(g[i] != nullptr, "parameter gradient of tensor %d without its gradient", i);
      MODDIT_CHECK_ARG(norm_kind != MODDIT_NORM_NONE && (j == 0 || norm_kind == MODDIT_NORM_LAYER),
                       "norm_kind %d has no such parameter", norm_kind);
    }
  MODDIT_CHECK_ARG((rope_cos == nullptr) == (rope_sin == nullptr), "rope_cos and rope_sin go together");
  if (rope_cos == nullptr) rope_form = MODDIT_ROPE_PAIR;
  if (norm_kind == MODDIT_NORM_RMS_ALL_HEADS)
    MODDIT_CHECK_ARG(static_cast<int64_t>(B) * S <= (1ll << 30), "B * S = %lld tokens are too many", static_cast<long long>(B) * S);
  if (rope_cos != nullptr) {
    MODDIT_CHECK_ARG(aligned16(rope_cos) && aligned16(rope_sin), "rotary tables must be 16-byte aligned");
    MODDIT_CHECK_ARG(0 <= rope_lo && rope_lo <= rope_hi && rope_hi <= S, "rotary range [%d, %d) outside 0..%d", rope_lo, rope_hi, S);
    MODDIT_CHECK_ARG(rope_form >= MODDIT_ROPE_ELEMENTWISE && rope_form <= MODDIT_ROPE_PAIR, "unknown rope_form %d", rope_form);
  }
  if (norm_kind == MODDIT_NORM_RMS_ALL_HEADS && width > kMaxWidth)
    return fail(MODDIT_E_UNSUPPORTED, "a normalisation over all heads covers at most %d values, got %lld", kMaxWidth,
                static_cast<long long>(width));
  if (any && (workspace == nullptr || !aligned16(workspace) || ws_bytes < moddit_qkv_prologue_bwd_workspace_bytes(B, S, H, D, norm_kind)))
    return fail(MODDIT_E_WORKSPACE, "parameter gradients need a 16-byte aligned workspace of %zu bytes",
                moddit_qkv_prologue_bwd_workspace_bytes(B, S, H, D, norm_kind));
  if (int rc = require_sm100()) return rc;

  const int blocks = blocks_for(B, S, H, D, norm_kind, dq != nullptr && dk != nullptr ? 2 : 1);
  const int64_t per = static_cast<int64_t>(blocks) * (norm_kind == MODDIT_NORM_RMS_ALL_HEADS ? width : 2 * D);
  BwdArgs a{};
  SumArgs sums{};
  for (int i = 0; i < 3; ++i) { a.g[i] = g[i]; a.dx[i] = dx[i]; }
  for (int i = 0; i < 2; ++i) {
    a.x[i] = x[i];
    a.part[i] = grads[i][0] || grads[i][1] ? static_cast<float*>(workspace) + i * per : nullptr;
    sums.part[i] = a.part[i];
    sums.out[i][0] = grads[i][0];
    sums.out[i][1] = grads[i][1];
  }
  a.weight[0] = q_weight; a.weight[1] = k_weight;
  a.cos = rope_cos; a.sin = rope_sin;
  a.token_stride = token_stride; a.out_stride = out_stride;
  a.B = B; a.S = S; a.H = H; a.N_out = N_out; a.src_row0 = src_row0;
  a.rope_form = rope_form; a.rope_lo = rope_lo; a.rope_hi = rope_hi;
  a.eps = eps;
  a.heads_per_item = heads_per_item(B, S, H, D);
  cudaStream_t st = as_stream(stream);
  if (dtype == MODDIT_BF16)
    return D == 128 ? launch_bwd<__nv_bfloat16, 128>(a, norm_kind, blocks, sums, st) : launch_bwd<__nv_bfloat16, 64>(a, norm_kind, blocks, sums, st);
  return D == 128 ? launch_bwd<__half, 128>(a, norm_kind, blocks, sums, st) : launch_bwd<__half, 64>(a, norm_kind, blocks, sums, st);
}
