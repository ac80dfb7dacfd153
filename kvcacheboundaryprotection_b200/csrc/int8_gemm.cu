// Matrix product in 8-bit integers with a scale for each token and each output channel:
//   y[m][n] = (sum_k xq[m][k] wq[n][k]) * sx[m] * sw[n] (+ bias[n])
// with exact 32-bit integer sums, and the per-token quantisation that feeds it.
#include <type_traits>

#include "common.cuh"
#include "kvbp_internal.h"

namespace kvbp {
namespace i8 {

// A row's codes from the bits m of its max|x|: rint(127 x / max|x|), every finite row.  The
// division works on x and max|x| times the power of two that brings max|x| to [1, 4) (a subnormal
// one to [2^-7, 1)): 127 x then neither overflows nor loses a bit, so half-way values are half-way
// (a value that the power of two makes subnormal is far below half a code).
struct RowQuant {
  float top, factor, up;
  bool fine;   // not zero, infinite or NaN: else every code is 0
  bool quick;  // 127 / top is finite
  __device__ __forceinline__ explicit RowQuant(uint32_t m) {
    top = __uint_as_float(m);
    fine = m > 0 && m < 0x7f800000u;
    quick = m >= 0x04000000u && m < 0x7f800000u;  // from 2^-119 on
    factor = quick ? 127.0f / top : 0.f;
    up = __uint_as_float((254u - min(max(m >> 23, 1u), 253u)) << 23);
  }
  __device__ __forceinline__ float scale() const { return top / 127.0f; }
  __device__ __forceinline__ uint32_t exact(float v) const {
    return fine ? static_cast<uint32_t>(static_cast<int>(rintf(127.0f * (v * up) / (top * up)))) : 0u;
  }
  // x times the rounded factor plus 1.5 * 2^23 leaves the integer in the low mantissa bits.  The
  // factor is off by 2^-24 of it, so a quotient (at most 127) by 8e-6: only what lies within
  // 1e-4 of half-way can round wrongly, and is divided.
  __device__ __forceinline__ uint2 eight(const uint4 w) const {
    const float x[8] = {bf16lo(w.x), bf16hi(w.x), bf16lo(w.y), bf16hi(w.y), bf16lo(w.z), bf16hi(w.z), bf16lo(w.w), bf16hi(w.w)};
    uint32_t c[8];
    float worst = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float s = fmaf(x[k], factor, 12582912.0f);
      worst = fmaxf(worst, fabsf(fmaf(x[k], factor, 12582912.0f - s)));
      c[k] = __float_as_uint(s);
    }
    if (!quick || worst > 0.4999f) {
#pragma unroll
      for (int k = 0; k < 8; ++k) c[k] = exact(x[k]);
    }
    auto bytes = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
      return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
    };
    return make_uint2(bytes(c[0], c[1], c[2], c[3]), bytes(c[4], c[5], c[6], c[7]));
  }
};
// m = max(m, max|x| of eight values) as bits: a NaN's bits are the largest
__device__ __forceinline__ uint32_t fold_max(uint32_t m, const uint4 w) {
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) m = max(m, max((ws[k] << 16) & 0x7fffffffu, ws[k] & 0x7fff0000u));
  return m;
}
__device__ __forceinline__ uint32_t abs_bits(const __nv_bfloat16 x) {
  return __float_as_uint(__bfloat162float(x)) & 0x7fffffffu;
}

// Per-token quantisation: sx = max|x| / 127 and the codes above (a zero row gives zeros and
// scale 0).  A row with a NaN or an infinity gets a scale that is not finite, and codes 0:
// every output of that token is then NaN.  One CTA per row, the row kept in registers between the
// maximum and the codes (kVec 16-byte vectors per thread: 2048 kVec values; what is beyond is read
// again, from L2).  Latency-bound: few registers let many rows share an SM.
template <int kVec>
__global__ void __launch_bounds__(256) quant_rows_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, int K,
                                                         int vec, int8_t* __restrict__ q, long long ldq,
                                                         float* __restrict__ scale) {
  pdl_wait();
  // only now: what runs before this kernel is complete when a dependent starts, so
  // kvbp_int8_linear's product may fetch weights before it waits for the codes
  pdl_launch_dependents();
  __shared__ uint32_t red[8];
  const size_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const __nv_bfloat16* row = x + r * ldx;
  int8_t* dst = q + r * ldq;
  const int nv = vec ? K / 8 : 0;
  const uint4* rv = reinterpret_cast<const uint4*>(row);
  uint4 keep[kVec];
  uint32_t m = 0;  // max|x| as bits: a NaN's bits are the largest
#pragma unroll
  for (int u = 0; u < kVec; ++u) {
    const int i = tid + 256 * u;
    keep[u] = i < nv ? rv[i] : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int u = 0; u < kVec; ++u) m = fold_max(m, keep[u]);
  for (int i = tid + 256 * kVec; i < nv; i += 256) m = fold_max(m, rv[i]);
  for (int i = nv * 8 + tid; i < K; i += 256) m = max(m, abs_bits(row[i]));
  m = __reduce_max_sync(0xffffffffu, m);
  if ((tid & 31) == 0) red[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = max(m, red[w]);
  const RowQuant rq(m);
  if (tid == 0) scale[r] = rq.scale();
  auto emit = [&](const uint4 w, int i) { *reinterpret_cast<uint2*>(dst + 8 * i) = rq.eight(w); };
#pragma unroll
  for (int u = 0; u < kVec; ++u) {
    const int i = tid + 256 * u;
    if (i < nv) emit(keep[u], i);
  }
  for (int i = tid + 256 * kVec; i < nv; i += 256) emit(rv[i], i);
  for (int i = nv * 8 + tid; i < K; i += 256) dst[i] = static_cast<int8_t>(rq.exact(__bfloat162float(row[i])));
}

// The same for rows of up to 1024: a warp per row, eight rows a CTA, no barrier.
__global__ void __launch_bounds__(256) quant_short_rows_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, int K,
                                                               int rows, int vec, int8_t* __restrict__ q, long long ldq,
                                                               float* __restrict__ scale) {
  pdl_wait();
  pdl_launch_dependents();  // as above
  const unsigned r = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= static_cast<unsigned>(rows)) return;
  const int lane = threadIdx.x & 31, nv = vec ? K / 8 : 0;
  const __nv_bfloat16* row = x + static_cast<size_t>(r) * ldx;
  int8_t* dst = q + static_cast<size_t>(r) * ldq;
  uint4 keep[4];
  uint32_t m = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    keep[u] = lane + 32 * u < nv ? reinterpret_cast<const uint4*>(row)[lane + 32 * u] : make_uint4(0, 0, 0, 0);
    m = fold_max(m, keep[u]);
  }
  for (int i = nv * 8 + lane; i < K; i += 32) m = max(m, abs_bits(row[i]));
  const RowQuant rq(__reduce_max_sync(0xffffffffu, m));
  if (lane == 0) scale[r] = rq.scale();
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (lane + 32 * u < nv) *reinterpret_cast<uint2*>(dst + 8 * (lane + 32 * u)) = rq.eight(keep[u]);
  for (int i = nv * 8 + lane; i < K; i += 32) dst[i] = static_cast<int8_t>(rq.exact(__bfloat162float(row[i])));
}

// ---- the product on the 5th-generation tensor cores (tcgen05.mma kind::i8) -------------
// The weight block is the M = 128 operand and the tokens the N = NT one, both K-major int8
// tiles of 128 bytes of K fetched by 2-D TMA with the 128-byte swizzle (rows and columns
// past the matrices arrive as zeros: sizes are free); the accumulator is int32 in TMEM, lane =
// output channel, column = token, so a warp's stores of one token's 32 channels are contiguous.
// Integer sums are exact, so K may be split and joined in any order with the same bits.
struct Args {
  const float* sw;
  const float* sx;
  const __nv_bfloat16* bias;
  void* out;
  long long ldo;
  int M, N, K, f32;
  const __nv_bfloat16* x;  // fused quantisation: the token itself
  int vec_x;  // it is 16-byte aligned
  int vec;    // four channels at a time are aligned
  int early;  // the weight is known to be complete before the kernel before this one ends
  int* err;
};

constexpr int kBK = 128;               // bytes (= codes) of K per stage: one swizzle atom
constexpr int kTileW = 128 * kBK;      // weight tile
constexpr int kMaxSplits = 8;          // a portable cluster
constexpr int kThreads = 6 * 32;       // producer, MMA, four epilogue warps

__host__ __device__ constexpr uint32_t idesc_i8(int N) {  // D s32, A and B s8, both K-major, M = 128
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_i8(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "l"(da), "l"(db), "r"(id), "r"(acc));
}
__device__ __forceinline__ int4 ld_dsmem_v4(uint32_t cluster_addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}
// sum * sx * sw + bias in fp32.  A token's scale beyond 2^64 comes last: sum * sx could overflow
// where the product with a small sw does not (sum * sw then overflows only where all of it does).
__device__ __forceinline__ bool far_scale(float sx) { return fabsf(sx) > 0x1p64f; }
__device__ __forceinline__ float scaled_sum(int sum, float sx, float sw, float bias, bool last) {
  return static_cast<float>(sum) * (last ? sw : sx) * (last ? sx : sw) + bias;
}
// scales and biases of channels n .. n + 3 (those below N)
struct Four {
  float sw[4], b[4];
  __device__ __forceinline__ void load(const Args& a, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sw[i] = n + i < a.N ? a.sw[n + i] : 0.f;
      b[i] = a.bias && n + i < a.N ? __bfloat162float(a.bias[n + i]) : 0.f;
    }
  }
  __device__ __forceinline__ void store(const Args& a, int m, int n, int4 acc, float sx) const {
    const bool far = far_scale(sx);
    const float y[4] = {scaled_sum(acc.x, sx, sw[0], b[0], far), scaled_sum(acc.y, sx, sw[1], b[1], far),
                        scaled_sum(acc.z, sx, sw[2], b[2], far), scaled_sum(acc.w, sx, sw[3], b[3], far)};
    const size_t at = static_cast<size_t>(m) * a.ldo + n;
    float* f = static_cast<float*>(a.out) + at;
    __nv_bfloat16* h = static_cast<__nv_bfloat16*>(a.out) + at;
    if (a.vec && n < a.N) {  // N, ldo multiples of 4, the output aligned
      if (a.f32) *reinterpret_cast<float4*>(f) = make_float4(y[0], y[1], y[2], y[3]);
      else *reinterpret_cast<uint2*>(h) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) {
        if (a.f32) f[i] = y[i];
        else h[i] = __float2bfloat16_rn(y[i]);
      }
  }
};
// Barrier among ``nthreads`` threads; true on all of them when ``v`` is on any.
__device__ __forceinline__ bool named_bar_or(int id, int nthreads, bool v) {
  uint32_t r;
  __syncwarp();  // the barrier wants whole warps; the waits before it may have split them
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\t"
      "bar.red.or.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(nthreads), "r"(static_cast<uint32_t>(v))
      : "memory");
  return r != 0;
}
// this thread's 16 or 32 accumulator columns from TMEM
template <int C>
__device__ __forceinline__ void ld_acc(uint32_t taddr, int (&v)[C]) {
  float f[C];
  if constexpr (C == 32) tc_ld32(taddr, f);
  else tc_ld16(taddr, f);
#pragma unroll
  for (int i = 0; i < C; ++i) v[i] = __float_as_int(f[i]);
}

// One output tile (128 channels x NT tokens) per cluster; the cluster's CTAs share the tile's
// K range (gridDim.x = cluster size) and join their int32 partial tiles over distributed shared
// memory.  Bound by the weight stream when tokens are few: stages are sized for two CTAs per SM.
// 16 tokens x 37888 x 3584: 25 us, 5.4 TB/s (quantisation: 2 us more); one token x 6144 x 2560:
// 6.9 us with its quantisation, 2.3 TB/s, latency.
// With kFuse (one token) the epilogue warps quantise the token themselves while the first
// weights are under way: each CTA reads all of x for its maximum (a few KB from L2) and puts its
// own K range's codes into shared memory as row 0 of the MMA's operand.  The other 15 rows hold
// anything: their columns of the accumulator are never stored.  That saves a launch: the GPU
// time is the same (6.9 against 7.4 us at 6144 x 2560, 27.7 against 26.5 at 37888 x 3584), the
// host's a third less.  (For four tokens the CTAs' repeated work cost more than the launch: 8.9
// against 7.5 us.)  The first weights wait for the kernel before this one, which may be the one
// that writes them; with more tokens the quantisation stands in between.
constexpr int kFuseSteps = 30;  // stages of K per CTA whose codes fit beside three of weights
template <int NT, bool kFuse>
struct Ring {
  static constexpr int kStage = kTileW + (kFuse ? 0 : NT * kBK);
  static constexpr int kStages = kFuse ? 3 : NT <= 32 ? 5 : NT == 64 ? 4 : 3;
  static constexpr int kTokens = kFuse ? kFuseSteps * NT * kBK : 0;
  static constexpr int kBytes = kStages * kStage + kTokens + 1024 + 256 + NT * 4 + 16;
  static_assert(kStages * kStage >= NT * 128 * 4, "the partial tile reuses the ring");
  static_assert(kBytes <= 115712, "two CTAs per SM");
};

template <int NT, bool kFuse>
__global__ void __launch_bounds__(kThreads, 2)
    split_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Args a) {
  using R = Ring<NT, kFuse>;
  constexpr int kCols = NT < 32 ? 32 : NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* tokens = base + R::kStages * R::kStage;  // kFuse: [step][16 rows][128], the token in row 0
  uint64_t* full = reinterpret_cast<uint64_t*>(tokens + R::kTokens);
  uint64_t* empty = full + R::kStages;
  uint64_t* done = empty + R::kStages;
  uint64_t* ready = done + 1;  // kFuse: the token's codes are in place
  uint32_t* tslot = reinterpret_cast<uint32_t*>(ready + 1);
  int* bad = reinterpret_cast<int*>(tslot + 1);
  float* sxs = reinterpret_cast<float*>(bad + 1);  // the tokens' scales
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = gridDim.x, rank = blockIdx.x;
  const int n0 = blockIdx.y * 128, m0 = blockIdx.z * NT;
  const int steps = (a.K + kBK - 1) / kBK;
  const int k0 = static_cast<int>(static_cast<long long>(rank) * steps / S);
  const int nk = static_cast<int>(static_cast<long long>(rank + 1) * steps / S) - k0;

  if (tid == 0) {
    for (int s = 0; s < R::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    mbar_init(ready, 128);
    *bad = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tslot;
  auto healthy = [&]() { return !*reinterpret_cast<volatile int*>(bad); };
  auto wait_or_fail = [&](uint64_t* bar, uint32_t ph) {
    if (mbar_wait_bounded(bar, ph)) return true;
    set_err(a.err, kErrWaitTimeout);
    atomicExch(bad, 1);
    return false;
  };

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&wmap);
      if (!kFuse) prefetch_tmap(&xmap);
      if (kFuse || !a.early) pdl_wait();
      auto load_w = [&](int u) {
        const int st = u % R::kStages;
        mbar_expect_tx(&full[st], R::kStage);
        tma_load_2d(base + st * R::kStage, &wmap, &full[st], (k0 + u) * kBK, n0);
      };
      auto load_x = [&](int u) {
        if (kFuse) return;
        const int st = u % R::kStages;
        tma_load_2d(base + st * R::kStage + kTileW, &xmap, &full[st], (k0 + u) * kBK, m0);
      };
      const int first = nk < R::kStages ? nk : R::kStages;
      for (int u = 0; u < first; ++u) load_w(u);
      if (!kFuse && a.early) pdl_wait();  // the tokens' codes come from the kernel before this one
      for (int u = 0; u < first; ++u) load_x(u);
      int issued = first;
      for (int u = first; u < nk && healthy(); ++u, ++issued) {
        if (!wait_or_fail(&empty[u % R::kStages], static_cast<uint32_t>(u / R::kStages - 1) & 1)) break;
        load_w(u);
        load_x(u);
      }
      pdl_launch_dependents();
      if (!healthy())  // let the copies in flight land before the CTA can exit
        for (int u = issued > R::kStages ? issued - R::kStages : 0; u < issued; ++u)
          mbar_wait_bounded(&full[u % R::kStages], static_cast<uint32_t>(u / R::kStages) & 1, 1u << 16);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      bool go = true;
      if (kFuse) {
        go = wait_or_fail(ready, 0);
        tc_after();
      }
      for (int u = 0; u < nk && go && healthy(); ++u) {
        const int st = u % R::kStages;
        if (!wait_or_fail(&full[st], static_cast<uint32_t>(u / R::kStages) & 1)) break;
        tc_after();
        const uint32_t sw = smem_u32(base + st * R::kStage);
        const uint32_t sx = kFuse ? smem_u32(tokens) + u * (NT * kBK) : sw + kTileW;
#pragma unroll
        for (int ks = 0; ks < kBK / 32; ++ks)
          mma_i8(tmem, tc_sdesc(sw + ks * 32), tc_sdesc(sx + ks * 32), idesc_i8(NT), (u > 0 || ks > 0) ? 1u : 0u);
        tc_commit(&empty[st]);
      }
      tc_commit(done);
    }
    __syncwarp();
  } else if (kFuse) {
    pdl_wait();
    uint32_t* red = reinterpret_cast<uint32_t*>(sxs + NT);  // the four warps' maxima
    const int et = tid - 64, nv = a.vec_x ? a.K / 8 : 0;
    const uint4* xv = reinterpret_cast<const uint4*>(a.x);
    uint32_t m = 0;
    for (int i = et; i < nv; i += 128) m = fold_max(m, xv[i]);
    for (int i = nv * 8 + et; i < a.K; i += 128) m = max(m, abs_bits(a.x[i]));
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) red[warp - 2] = m;
    __syncwarp();
    named_bar(1, 128);
    const RowQuant rq(max(max(red[0], red[1]), max(red[2], red[3])));
    if (et == 0) sxs[0] = rq.scale();
    for (int c = et; c < nk * 16; c += 128) {  // eight codes at a time of this CTA's K range
      const int k = k0 * kBK + 8 * c;          // columns past K meet zero weights
      uint2 codes = make_uint2(0, 0);
      if (k / 8 < nv) {
        codes = rq.eight(xv[k / 8]);
      } else if (k < a.K) {
        uint32_t b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = k + i < a.K ? rq.exact(__bfloat162float(a.x[k + i])) & 255u : 0u;
        codes = make_uint2(b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24, b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24);
      }
      *reinterpret_cast<uint2*>(tokens + (c >> 4) * (NT * kBK) + (c & 15) * 8) = codes;  // row 0 has no swizzle
    }
    fence_proxy_async_smem();
    mbar_arrive(ready);
  }
  const bool ok = wait_or_fail(done, 0) && healthy();
  __syncwarp();
  tc_after();
  pdl_wait();  // before the scales are read and anything is written
  const int cols = min(NT, a.M - m0);  // live tokens of the tile
  if (!kFuse && tid < cols) sxs[tid] = a.sx[m0 + tid];
  const bool all_ok = !__syncthreads_or(!ok);
  // The accumulator goes through shared memory (the drained ring), [token][128 channels], so
  // that the stores are 8 or 16 bytes a thread and run along the channels.  (Stored straight
  // from TMEM, one channel a lane, the 128-token tile took 11 us for its 16 KiB.)
  int* part = reinterpret_cast<int*>(base);
  if (warp >= 2 && all_ok) {
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    int* mine = part + q * 32 + lane;
    const uint32_t acc = tmem + (static_cast<uint32_t>(q * 32) << 16);
    constexpr int C = NT < 32 ? 16 : 32;
#pragma unroll 1
    for (int c = 0; c < cols; c += C) {
      int v[C];
      ld_acc<C>(acc + c, v);
#pragma unroll
      for (int i = 0; i < C; ++i) mine[(c + i) * 128] = v[i];
    }
  }
  if (S > 1) cluster_sync_all();
  else __syncthreads();
  // this CTA's share of the tile's live elements, four channels at a time
  const int E = cols * 32, e1 = static_cast<int>(static_cast<long long>(rank + 1) * E / S);
  if (all_ok) {
    const int e0 = static_cast<int>(static_cast<long long>(rank) * E / S) + tid;
    const int n = n0 + (e0 & 31) * 4;  // the same in every turn: kThreads is a multiple of 32
    Four four;
    four.load(a, n);
#pragma unroll 2
    for (int e = e0; e < e1; e += kThreads) {
      int4 sum = make_int4(0, 0, 0, 0);
      if (S > 1) {
        const uint32_t at = smem_u32(part + 4 * e);
        int4 v[kMaxSplits];  // all peers' values before the first addition
#pragma unroll
        for (int r = 0; r < kMaxSplits; ++r) v[r] = r < S ? ld_dsmem_v4(mapa_u32(at, r)) : make_int4(0, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < kMaxSplits; ++r) sum.x += v[r].x, sum.y += v[r].y, sum.z += v[r].z, sum.w += v[r].w;
      } else {
        sum = *reinterpret_cast<const int4*>(part + 4 * e);
      }
      four.store(a, m0 + (e >> 5), n, sum, sxs[e >> 5]);
    }
  }
  if (S > 1) cluster_sync_all();  // no CTA leaves while a peer may still read its part
  tc_before();
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
}

// Many tokens: persistent, one CTA per SM over 128 x 256 tiles in a grouped raster, a ring of
// four 48 KiB stages that runs on across tiles, and two accumulators in TMEM so that the MMAs
// of one tile run while the epilogue warps drain the other.  8192 x 37888 x 3584 with its
// quantisation: 830 us, 2.7 POP/s, a dozen at a time; 925 us held up at the power limit; per stage
// and SM 48 KiB from L2.
constexpr int kPN = 256;
constexpr int kPStages = 4;
constexpr int kPStage = kTileW + kPN * kBK;
constexpr int kPBytes = kPStages * kPStage + 1024 + 256 + 2 * kPN * 4;
constexpr int kPEpilogue = 16;  // warps: with four, one a scheduler, a tile's 256 tokens took 8 us
constexpr int kPThreads = (2 + kPEpilogue) * 32;
constexpr int kBand = 16;  // channel tiles per raster band (4 to 64 within 2 % of it at 8192 x 37888 x 3584)

__global__ void __launch_bounds__(kPThreads, 1)
    persist_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sxs = reinterpret_cast<float*>(base + kPStages * kPStage);  // [2][kPN] token scales of a tile
  uint64_t* full = reinterpret_cast<uint64_t*>(sxs + 2 * kPN);
  uint64_t* empty = full + kPStages;
  uint64_t* accfull = empty + kPStages;
  uint64_t* accempty = accfull + 2;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(accempty + 2);
  int* bad = reinterpret_cast<int*>(tslot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tn = (a.N + 127) / 128, tm = (a.M + kPN - 1) / kPN;
  const long long tiles = static_cast<long long>(tn) * tm;
  const int steps = (a.K + kBK - 1) / kBK;
  // tile t: bands of kBand channel tiles, tokens the slow index within a band
  auto tile_of = [&](long long t, int& n0, int& m0) {
    const long long per = static_cast<long long>(kBand) * tm;
    const int band = static_cast<int>(t / per);
    const int in = static_cast<int>(t - band * per), width = min(kBand, tn - band * kBand);
    n0 = (band * kBand + in % width) * 128;
    m0 = in / width * kPN;
  };
  if (tid == 0) {
    for (int s = 0; s < kPStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accfull[b], 1);
      mbar_init(&accempty[b], kPEpilogue);
    }
    *bad = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(2 * kPN));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tslot;
  auto healthy = [&]() { return !*reinterpret_cast<volatile int*>(bad); };
  auto wait_or_fail = [&](uint64_t* bar, uint32_t ph) {
    if (mbar_wait_bounded(bar, ph)) return true;
    set_err(a.err, kErrWaitTimeout);
    atomicExch(bad, 1);
    return false;
  };
  pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&wmap);
      prefetch_tmap(&xmap);
      long long g = 0;
      for (long long t = blockIdx.x; t < tiles && healthy(); t += gridDim.x) {
        int n0, m0;
        tile_of(t, n0, m0);
        for (int u = 0; u < steps; ++u, ++g) {
          const int st = static_cast<int>(g % kPStages);
          if (g >= kPStages && !wait_or_fail(&empty[st], static_cast<uint32_t>(g / kPStages - 1) & 1)) break;
          if (!healthy()) break;
          mbar_expect_tx(&full[st], kPStage);
          tma_load_2d(base + st * kPStage, &wmap, &full[st], u * kBK, n0);
          tma_load_2d(base + st * kPStage + kTileW, &xmap, &full[st], u * kBK, m0);
        }
      }
      pdl_launch_dependents();
      if (!healthy())
        for (long long u = g > kPStages ? g - kPStages : 0; u < g; ++u)
          mbar_wait_bounded(&full[u % kPStages], static_cast<uint32_t>(u / kPStages) & 1, 1u << 16);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      long long g = 0;
      int i = 0;
      for (long long t = blockIdx.x; t < tiles && healthy(); t += gridDim.x, ++i) {
        const int buf = i & 1;
        if (i >= 2 && !wait_or_fail(&accempty[buf], static_cast<uint32_t>((i >> 1) - 1) & 1)) break;
        tc_after();
        const uint32_t acc = tmem + static_cast<uint32_t>(buf * kPN);
        bool ok = true;
        for (int u = 0; u < steps; ++u, ++g) {
          const int st = static_cast<int>(g % kPStages);
          if (!wait_or_fail(&full[st], static_cast<uint32_t>(g / kPStages) & 1)) {
            ok = false;
            break;
          }
          tc_after();
          const uint32_t sw = smem_u32(base + st * kPStage), sx = sw + kTileW;
#pragma unroll
          for (int ks = 0; ks < kBK / 32; ++ks)
            mma_i8(acc, tc_sdesc(sw + ks * 32), tc_sdesc(sx + ks * 32), idesc_i8(kPN), (u > 0 || ks > 0) ? 1u : 0u);
          tc_commit(&empty[st]);
        }
        if (!ok) break;
        tc_commit(&accfull[buf]);
      }
    }
    __syncwarp();
  } else {
    // four warps per TMEM lane quarter, a quarter of the tokens each
    constexpr int kShare = kPN * 4 / kPEpilogue;
    const int q = warp & 3, et = tid - 64, share = (warp - 2) / 4 * kShare;
    int i = 0;
    for (long long t = blockIdx.x; t < tiles; t += gridDim.x, ++i) {
      const int buf = i & 1;
      int n0, m0;
      tile_of(t, n0, m0);
      const int n = n0 + q * 32 + lane, cols = min(kPN, a.M - m0);
      for (int c = et; c < kPN; c += kPEpilogue * 32) sxs[buf * kPN + c] = c < cols ? a.sx[m0 + c] : 0.f;
      const bool ok = wait_or_fail(&accfull[buf], static_cast<uint32_t>(i >> 1) & 1);
      tc_after();
      // the tile's scales are in place, and all epilogue warps leave together after a failed wait
      if (named_bar_or(1, kPEpilogue * 32, !ok || !healthy())) break;
      const uint32_t acc = tmem + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(buf * kPN);
      const float* sx = sxs + buf * kPN;
      // one channel a lane; the warp reads TMEM as a whole, past the last channel too
      const bool in = n < a.N;
      const float sw = in ? a.sw[n] : 0.f, bias = a.bias && in ? __bfloat162float(a.bias[n]) : 0.f;
      const size_t row = static_cast<size_t>(m0 + share) * a.ldo + n;
      float* pf = static_cast<float*>(a.out) + row;
      __nv_bfloat16* ph = static_cast<__nv_bfloat16*>(a.out) + row;
#pragma unroll 1
      for (int c = share; c < min(cols, share + kShare); c += 32) {
        int v[32];
        __syncwarp();
        ld_acc<32>(acc + c, v);
        const int live = in ? cols - c : 0;
        auto put = [&](auto some_far) {
          auto y = [&](int k) {
            return scaled_sum(v[k], sx[c + k], sw, bias, decltype(some_far)::value && far_scale(sx[c + k]));
          };
          if (a.f32) {
#pragma unroll
            for (int k = 0; k < 32; ++k, pf += a.ldo)
              if (k < live) *pf = y(k);
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k, ph += a.ldo)
              if (k < live) *ph = __float2bfloat16_rn(y(k));
          }
        };
        // asked once for the 32 tokens: the comparison for each sum cost 1.2 % of the large product
        if (__any_sync(0xffffffffu, far_scale(sx[c + lane]))) put(std::true_type{});
        else put(std::false_type{});
      }
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&accempty[buf]);
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * kPN));
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// An int8 matrix [rows][ld] as tiles of ``box`` rows x 128 columns, 128-byte swizzled.
static CUresult tile_map(CUtensorMap* map, const void* p, int rows, int K, long long ld, int box) {
  static EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<EncodeTiledFn>(ptr);
  }();
  if (!fn) return CUDA_ERROR_NOT_FOUND;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t boxes[2] = {kBK, static_cast<cuuint32_t>(box)};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, boxes, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

template <int NT, bool kFuse>
static cudaError_t launch_split(cudaStream_t st, const CUtensorMap& wm, const CUtensorMap& xm, const Args& a, int S) {
  constexpr int smem = Ring<NT, kFuse>::kBytes;
  if (prepare_device(reinterpret_cast<const void*>(split_kernel<NT, kFuse>), smem) <= 0) return cudaErrorNoDevice;
  const dim3 grid(S, (a.N + 127) / 128, (a.M + NT - 1) / NT);
  return launch_pdl(split_kernel<NT, kFuse>, grid, dim3(kThreads), smem, st, S > 1 ? dim3(S, 1, 1) : dim3(0), wm, xm, a);
}

static int quant_rows(cudaStream_t st, int rows, int K, const void* x, long long ldx, void* q, long long ldq, float* scale) {
  if (!x || !q || !scale) return fail(kStatusArg, "int8_quant_rows: null pointer");
  if (rows <= 0 || K <= 0 || ldx < K || ldq < K) return fail(kStatusArg, "int8_quant_rows: bad size");
  if (misaligned(q, 16) || ldq % 16) return fail(kStatusArg, "int8_quant_rows: q rows must be 16-byte aligned");
  // 16-byte loads where x's rows allow them, else one value at a time
  const int vec = !misaligned(x, 16) && ldx % 8 == 0;
  const __nv_bfloat16* xb = static_cast<const __nv_bfloat16*>(x);
  int8_t* qb = static_cast<int8_t*>(q);
  cudaError_t e;
  // Short rows a warp each, for many rows (8192 of 128: 4.4 us against 12.3, of 1024: 7.9 against
  // 14.4; few rows lose up to a microsecond: 300 of 1024 3.1 against 2.0).  Longer ones a CTA each
  // with as few vectors in registers as pays, since many rows then share an SM (8192 rows, two
  // vectors against five: K = 4096 26 us and 35, 6144 40 and 42, 8192 52 and 48, 10240 64 and 55);
  // past 10240 reading most of the row twice is faster than eight vectors (12288 64 us against 75,
  // 18944 100 against 125).
  if (K <= 1024) {
    e = launch_pdl(quant_short_rows_kernel, dim3((static_cast<unsigned>(rows) + 7) / 8), dim3(256), 0, st, dim3(0), xb, ldx,
                   K, rows, vec, qb, ldq, scale);
  } else {
    auto kernel = K > 6144 && K <= 10240 ? quant_rows_kernel<5> : quant_rows_kernel<2>;
    e = launch_pdl(kernel, dim3(rows), dim3(256), 0, st, dim3(0), xb, ldx, K, vec, qb, ldq, scale);
  }
  if (e != cudaSuccess) return fail(kStatusCuda, "int8_quant_rows launch: %s", cudaGetErrorString(e));
  return kStatusOk;
}

// CTAs that share a tile's K range: two per SM but for a seventh of them (larger clusters do not
// fill the last places: 72 tiles of 200 tokens took 19.2 us in 4 parts, 288 CTAs, and 14.3 us in
// 3; pairs do: 144 tiles of 512 tokens 17.9 us in 2, 21.1 unsplit), each with at least four
// stages of K, within a portable cluster.
static int room(int sms) { return 2 * sms * 6 / 7; }
static int splits(long long tiles, int steps, int sms) {
  long long s = room(sms) / tiles;
  if (s < 2 && tiles <= sms) s = 2;
  if (s > steps / 4) s = steps / 4;
  return s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : static_cast<int>(s);
}

static long long out_bytes(const Args& a) { return ((a.M - 1ll) * a.ldo + a.N) * (a.f32 ? 4 : 2); }

// Checks of all but the tokens.
static int check(const Args& a, const void* w, long long ldw) {
  if (!w || !a.sw || !a.out) return fail(kStatusArg, "int8_gemm: null pointer");
  if (a.M <= 0 || a.N <= 0 || a.K <= 0 || ldw < a.K || a.ldo < a.N) return fail(kStatusArg, "int8_gemm: bad size");
  // the sum of K products of up to 127 * 128 stays in 32 bits
  if (a.K > 131071) return fail(kStatusUnsupported, "int8_gemm: K %d > 131071 could overflow the 32-bit sums", a.K);
  if (misaligned(w, 16) || ldw % 16) return fail(kStatusArg, "int8_gemm: w's rows must be 16-byte aligned");
  if (misaligned(a.out, a.f32 ? 4 : 2)) return fail(kStatusArg, "int8_gemm: misaligned output");
  if (a.N > 65535 * 128 || a.M > 0x7ffffe00) return fail(kStatusUnsupported, "int8_gemm: M %d or N %d is too large", a.M, a.N);
  if (overlap(a.out, out_bytes(a), w, (a.N - 1ll) * ldw + a.K)) return fail(kStatusArg, "int8_gemm: out must not overlap w");
  return kStatusOk;
}

static int gemm(cudaStream_t st, Args a, const void* w, long long ldw, const void* xq, long long ldq) {
  if (int bad = check(a, w, ldw)) return bad;
  if (!xq || !a.sx) return fail(kStatusArg, "int8_gemm: null pointer");
  if (ldq < a.K) return fail(kStatusArg, "int8_gemm: bad size");
  if (misaligned(xq, 16) || ldq % 16) return fail(kStatusArg, "int8_gemm: xq's rows must be 16-byte aligned");
  if (overlap(a.out, out_bytes(a), xq, (a.M - 1ll) * ldq + a.K)) return fail(kStatusArg, "int8_gemm: out must not overlap xq");
  a.vec = a.N % 4 == 0 && a.ldo % 4 == 0 && !misaligned(a.out, a.f32 ? 16 : 8);
  const int sms = prepare_device(reinterpret_cast<const void*>(persist_kernel), kPBytes);
  if (sms <= 0) return fail(kStatusCuda, "int8_gemm: no usable CUDA device");
  const long long tn = (a.N + 127) / 128;
  const int steps = (a.K + kBK - 1) / kBK;
  // The persistent form from half a wave of its tiles on (1024 x 2560 x 2560, 80 tiles: 15.8 us
  // against 19.0; 512 x 4608 x 3584, 72 tiles: 18.3 against 17.9).  Below, the narrowest tile that
  // holds the tokens, but 64 twice instead of 128 where that leaves room to split K (128 x 2560 x
  // 9728: 15.1 us against 16.4; without room, 128 x 37888 x 3584: 60 against 39).
  const bool many = a.M > 128 && tn * ((a.M + kPN - 1) / kPN) * 2 > sms;
  const int NT = many ? kPN : a.M <= 16 ? 16 : a.M <= 32 ? 32 : a.M <= 64 || (a.M <= 128 && tn * 4 <= room(sms)) ? 64 : 128;
  const long long tm = (a.M + NT - 1) / NT;
  if (!many && tm > 65535) return fail(kStatusUnsupported, "int8_gemm: too many tiles");
  CUtensorMap wm, xm;
  CUresult r = tile_map(&wm, w, a.N, a.K, ldw, 128);
  if (r == CUDA_SUCCESS) r = tile_map(&xm, xq, a.M, a.K, ldq, NT);
  if (r != CUDA_SUCCESS) return fail(kStatusCuda, "int8_gemm: tensor map failed (%d)", static_cast<int>(r));
  const int S = splits(tn * tm, steps, sms);
  cudaError_t e;
  if (many)
    e = launch_pdl(persist_kernel, dim3(static_cast<unsigned>(tn * tm < sms ? tn * tm : sms)), dim3(kPThreads), kPBytes, st, dim3(0), wm, xm, a);
  else if (NT == 16)
    e = launch_split<16, false>(st, wm, xm, a, S);
  else if (NT == 32)
    e = launch_split<32, false>(st, wm, xm, a, S);
  else if (NT == 64)
    e = launch_split<64, false>(st, wm, xm, a, S);
  else
    e = launch_split<128, false>(st, wm, xm, a, S);
  if (e != cudaSuccess) return fail(kStatusCuda, "int8_gemm launch: %s", cudaGetErrorString(e));
  return kStatusOk;
}

// One token straight from bf16: quantisation and product in one kernel.
static bool fused(int M, int K) { return M == 1 && K <= kFuseSteps * kMaxSplits * kBK; }

static int gemm_fused(cudaStream_t st, Args a, const void* w, long long ldw) {
  a.vec = a.N % 4 == 0 && a.ldo % 4 == 0 && !misaligned(a.out, a.f32 ? 16 : 8);
  a.vec_x = !misaligned(a.x, 16);
  const int sms = prepare_device(reinterpret_cast<const void*>(split_kernel<16, true>), Ring<16, true>::kBytes);
  if (sms <= 0) return fail(kStatusCuda, "int8_linear: no usable CUDA device");
  CUtensorMap wm;
  const CUresult r = tile_map(&wm, w, a.N, a.K, ldw, 128);
  if (r != CUDA_SUCCESS) return fail(kStatusCuda, "int8_linear: tensor map failed (%d)", static_cast<int>(r));
  const int steps = (a.K + kBK - 1) / kBK, least = (steps + kFuseSteps - 1) / kFuseSteps;
  const int S = splits((a.N + 127) / 128, steps, sms);
  const cudaError_t e = launch_split<16, true>(st, wm, wm, a, S < least ? least : S);
  if (e != cudaSuccess) return fail(kStatusCuda, "int8_linear launch: %s", cudaGetErrorString(e));
  return kStatusOk;
}

}  // namespace i8
}  // namespace kvbp

#include "../../include/kvbp.h"

extern "C" int kvbp_int8_quant_rows(kvbp_stream_t stream, int32_t rows, int32_t K, const void* x, int64_t ldx, void* q,
                                    int64_t ldq, float* scale) {
  return kvbp::i8::quant_rows(reinterpret_cast<cudaStream_t>(stream), rows, K, x, ldx, q, ldq, scale);
}

extern "C" int kvbp_int8_gemm(kvbp_stream_t stream, int32_t fp32_out, int32_t M, int32_t N, int32_t K, const void* w,
                              int64_t ldw, const float* w_scale, const void* xq, int64_t ldq, const float* x_scale,
                              const void* bias, void* out, int64_t ldo, int32_t* dev_err) {
  const kvbp::i8::Args a{w_scale, x_scale, static_cast<const __nv_bfloat16*>(bias), out, ldo, M, N, K, fp32_out ? 1 : 0, nullptr, 0, 0, 0, dev_err};
  return kvbp::i8::gemm(reinterpret_cast<cudaStream_t>(stream), a, w, ldw, xq, ldq);
}

extern "C" int64_t kvbp_int8_linear_workspace(int32_t M, int32_t K) {
  if (M <= 0 || K <= 0 || kvbp::i8::fused(M, K)) return 0;
  return static_cast<int64_t>(M) * ((static_cast<int64_t>(K) + 15) / 16 * 16) + 4ll * M;
}

extern "C" int kvbp_int8_linear(kvbp_stream_t stream, int32_t fp32_out, int32_t M, int32_t N, int32_t K, const void* w,
                                int64_t ldw, const float* w_scale, const void* x, int64_t ldx, const void* bias,
                                void* out, int64_t ldo, void* workspace, int64_t workspace_bytes, int32_t* dev_err) {
  kvbp::i8::Args a{w_scale, nullptr, static_cast<const __nv_bfloat16*>(bias), out, ldo, M, N, K, fp32_out ? 1 : 0,
                   static_cast<const __nv_bfloat16*>(x), 0, 0, 1, dev_err};
  // the product's arguments first: a refused call leaves the workspace alone
  if (int st = kvbp::i8::check(a, w, ldw)) return st;
  if (!x || ldx < K) return kvbp::fail(kvbp::kStatusArg, "int8_linear: bad x");
  if (kvbp::overlap(out, kvbp::i8::out_bytes(a), x, 2 * ((M - 1ll) * ldx + K)))
    return kvbp::fail(kvbp::kStatusArg, "int8_linear: out must not overlap x");
  if (kvbp::i8::fused(M, K)) return kvbp::i8::gemm_fused(reinterpret_cast<cudaStream_t>(stream), a, w, ldw);
  if (!workspace || kvbp::misaligned(workspace, 16)) return kvbp::fail(kvbp::kStatusArg, "int8_linear: no aligned workspace");
  if (workspace_bytes < kvbp_int8_linear_workspace(M, K))
    return kvbp::fail(kvbp::kStatusArg, "int8_linear: workspace of %lld bytes is too small", static_cast<long long>(workspace_bytes));
  const int64_t ldq = (static_cast<int64_t>(K) + 15) / 16 * 16;
  float* scale = reinterpret_cast<float*>(static_cast<char*>(workspace) + ldq * M);
  if (int st = kvbp_int8_quant_rows(stream, M, K, x, ldx, workspace, ldq, scale)) return st;
  a.sx = scale;
  return kvbp::i8::gemm(reinterpret_cast<cudaStream_t>(stream), a, w, ldw, workspace, ldq);
}
