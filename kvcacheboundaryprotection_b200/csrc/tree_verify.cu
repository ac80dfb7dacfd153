// Verification of drafted tokens against the target's probabilities (speculative decoding).
//
// One walk over a sequence's nodes j = 1 .. T-1 in order: a node whose parent is the last
// accepted node is tested.  With r the target's weights at that parent (what earlier siblings
// left of them), R their sum, x the node's token and q the distribution that x was drawn from
// (1 at x where there is none), the node is accepted when u * q(x) * R < r(x); otherwise
//   r <- max(r / R - q, 0)        (r(x) <- 0 where q is 1 at x).
// Each test keeps the target's law, x being an independent draw from q: P(accept x) + the residual's mass
// add up to r / R.  The last accepted node's r gives one more token: the first x whose running sum exceeds u * R.
//
// A token is chosen where a running sum of a hundred thousand terms passes a border; it has to be the
// token that the definition gives, so sums in 32 bits are trusted only as far as their error goes:
// every node's row is read once with fp32 weights, whose sums are off by less than ``eps`` of the row's; a
// test or a draw that comes out the same anywhere within that is decided, another one is made again with
// double weights (one in some ten thousand tests, and draws that end in a flat tail).  A random draft's
// residuals, differences of near values, carry a bound of their own that grows with every rejection.
//
// A cluster of CTAs per sequence, each with a contiguous share of the row, each warp with a contiguous
// share of that: a warp's sum is both part of the row's and, for the draw, the sum of what lies before the
// next one's.  The CTAs exchange their sums through shared memory and take every decision alike.
//
// What bounds it is the chain of a path: a row is 2.3 us of loads and 2 of joins (warps, CTAs), and the next
// row is known only then.  On B200 (graph replay on the same inputs, the smaller ones in L2): greedy 16 x 16 nodes x 152064 tokens, five levels: 25 us; one
// sequence with a draft's distributions, two levels, a rejection and the draw: 28 us; 64 x 32 nodes with them:
// 160 to 500 us with the inputs, the time of the sequence with the most rejections.
#include <math.h>

#include "common.cuh"
#include "kvbp_internal.h"

namespace kvbp {
namespace tv {

constexpr int kMaxNodes = 128;
constexpr int kMaxCluster = 8;
constexpr int kNone = 0x7fffffff;

struct Args {
  int T, V;
  const void* target;
  long long ldt;
  const float* temperature;
  const int* tokens;
  const int* parents;
  const float* draft;
  long long ldd;
  const float* accept_u;
  const float* sample_u;
  int* path;
  int* n_path;
  int* next_token;
  int* err;
};

// maximum of three, NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename L>
struct Row;
template <>
struct Row<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void many(const uint4& v, float (&x)[8]) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  }
};
template <>
struct Row<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void many(const uint4& v, float (&x)[8]) {
    x[0] = bf16lo(v.x), x[1] = bf16hi(v.x), x[2] = bf16lo(v.y), x[3] = bf16hi(v.y);
    x[4] = bf16lo(v.z), x[5] = bf16hi(v.z), x[6] = bf16lo(v.w), x[7] = bf16hi(v.w);
  }
};

// What one CTA tells the others: its largest logit and the first index of it, its sum relative to that;
// or a double sum.
struct alignas(16) Message {
  float top;
  int first;
  double sum;
};

// e^y, y <= 0, by Tang's table-driven method (ACM TOMS 15, 1989): y = n ln2 / 32 + r, e^r by its series,
// 2^(n / 32) from a table.  |r| <= ln2 / 64, so that the series' rest r^6 / 720 is below 3e-15; the reduction by
// one rounded constant adds 2^-53 |y|.
__device__ __forceinline__ double exp_of(double y, const double* table) {
  if (!(y > -700.0)) return 0.0;
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: the nearest integer is left in the low bits
  const double t = fma(y, 46.166241308446828384, kRound);  // 32 / ln 2
  const int n = __double2loint(t);
  const double r = fma(t - kRound, -0.021660849392498290195, y);  // ln 2 / 32
  double p = fma(r, 1.0 / 120, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const double v = table[n & 31] * p;
  return __hiloint2double(__double2hiint(v) + (n >> 5) * (1 << 20), __double2loint(v));
}

// kThreads: 512, or 256 where two CTAs share an SM.  (128 registers a thread either way: at 64 the spills cost
// more than the second CTA gains.)
template <typename L, int kThreads>
__global__ void __launch_bounds__(kThreads, 512 / kThreads) verify_kernel(Args a) {
  constexpr int kWarps = kThreads / 32;
  using R = Row<L>;
  constexpr int N = R::N;
  __shared__ Message box[2];
  __shared__ float w_top[kWarps];
  __shared__ int w_first[kWarps];
  __shared__ double s_part[kWarps];
  __shared__ double w_sum[kWarps];  // each warp's sum at the current node, relative to ``top``
  __shared__ double s_R[kMaxNodes + 1], s_inv[kMaxNodes + 1];  // sums after 0, 1, ... rejections
  __shared__ float s_finv[kMaxNodes + 1];
  __shared__ int s_rej[kMaxNodes];
  __shared__ int s_par[kMaxNodes], s_tok[kMaxNodes];
  __shared__ float s_u[kMaxNodes];
  __shared__ double table[32];
  __shared__ __align__(8) int s_token[2];  // the draw: token, and whether it is certain
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float NEG_INF = -__int_as_float(0x7f800000);
  uint32_t rank, cs;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(cs));
  const int b = blockIdx.x / cs;
  if (tid < 32) table[tid] = exp2(tid / 32.0);
  pdl_launch_dependents();
  pdl_wait();
  const int T = a.T, V = a.V;
  for (int i = tid; i < T; i += kThreads) {
    s_par[i] = a.parents[static_cast<size_t>(b) * T + i];
    s_tok[i] = a.tokens[static_cast<size_t>(b) * T + i];
    s_u[i] = a.accept_u[static_cast<size_t>(b) * T + i];
  }
  const float heat = a.temperature ? a.temperature[b] : 1.f;
  const float draw = a.sample_u[b];
  __syncthreads();
  int* path = a.path + static_cast<size_t>(b) * T;
  const bool greedy = !(heat > 0.f);
  const double inv = 1.0 / static_cast<double>(greedy ? 1.f : heat);
  const float c = static_cast<float>(1.4426950408889634 * inv);
  if (s_par[0] != -1) {  // no tree
    if (rank == 0) {
      for (int i = tid; i < T; i += kThreads) {
        path[i] = -1;
        if (s_par[i] >= i) set_err(a.err, kErrIndex);
      }
      if (tid == 0) {
        a.n_path[b] = 0;
        a.next_token[b] = -1;
      }
    }
    return;  // the whole cluster does
  }
  const bool drawn = a.draft && !greedy;
  const L* row = nullptr;
  const float* q = nullptr;
  // this warp's share of the row: the head up to the first 16-byte boundary (first warp), vectors
  // [lo, hi), the tail (last warp)
  int head = 0, tail = 0, lo = 0, hi = 0;
  int parity = 0, n_rej = 0, first = kNone;
  float top = NEG_INF;
  double S = 0.0;      // the row's sum in fp32 weights
  float base_eps = 0.f, eps = 0.f, sum_eps = 0.f;  // (sum_eps: the summation's part)
  bool odd_row = false;  // NaN or infinities decide: no short cuts
  double E = 0.0;  // how far the weights that the rejections of a random draft left may be off, all together
  bool exact = false;  // s_R and w_sum are double sums

  auto share = [&]() {
    const int ahead = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(L));
    head = min(V, ahead);
    const int vecs = (V - head) / N;
    tail = V - head - vecs * N;
    const int w = rank * kWarps + warp, all = cs * kWarps;
    lo = static_cast<int>(static_cast<long long>(vecs) * w / all);
    hi = static_cast<int>(static_cast<long long>(vecs) * (w + 1) / all);
    if (w != 0) head = 0;
    if (w != all - 1) tail = 0;
    // error of the row's fp32 sum: the weights' (2^x of the hardware 2^-22; the exponent's roundings, 2^-24 of
    // up to 31, beyond which a row's terms do not matter, and of the maximum's, below) and the joins': 24 steps of 2^-22;
    // for each vector of a lane its sums and one change of the reference maximum: 3 steps
    sum_eps = (16.f + static_cast<float>(vecs / (all * 32) + 1)) * 0x1p-24f;
    base_eps = (24.f + 3.f * static_cast<float>(vecs / (all * 32) + 1)) * 0x1p-22f;
  };
  auto vec0 = [&]() { return min(V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(L))); };
  auto clean = [&](float l) { return l == l ? l : NEG_INF; };

  auto sync_cluster = []() {
    __syncwarp();  // (the cluster's barrier wants whole warps)
    cluster_sync_all();
  };

  // ---- double weights
  auto weight = [&](float l) -> double {
    if (l == top) return 1.0;
    return l < top ? exp_of((static_cast<double>(l) - static_cast<double>(top)) * inv, table) : 0.0;
  };
  auto rest_of = [&](int x, float l, float qx) -> double {  // what the rejections left of token x
    if (greedy) return x == first ? 1.0 : 0.0;
    double r = weight(l);
    if (drawn) {
      for (int j = 0; j < n_rej; ++j) r = fmax(fma(r, s_inv[j], -static_cast<double>(qx)), 0.0);
    } else {
      for (int j = 0; j < n_rej; ++j)
        if (x == s_rej[j]) r = 0.0;
    }
    return r;
  };
  auto rest = [&](int x, float l) -> double { return rest_of(x, l, drawn && n_rej ? q[x] : 0.f); };
  auto rest_fast = [&](int x, float l) -> float {  // the same with fp32 weights
    float r = l == top ? 1.f : ex2((l - top) * c);
    if (drawn) {
      if (n_rej) {
        const float qx = q[x];
        for (int j = 0; j < n_rej; ++j) r = fmaxf(fmaf(r, s_finv[j], -qx), 0.f);
      }
    } else {
      for (int j = 0; j < n_rej; ++j)
        if (x == s_rej[j]) r = 0.f;
    }
    return r;
  };
  // the elements [from, to) of warp w of all the cluster's
  auto range = [&](int w, int& from, int& to) {
    const int v0 = vec0(), vecs = (V - v0) / N, all = cs * kWarps;
    from = w == 0 ? 0 : v0 + static_cast<int>(static_cast<long long>(vecs) * w / all) * N;
    to = w == all - 1 ? V : v0 + static_cast<int>(static_cast<long long>(vecs) * (w + 1) / all) * N;
  };
  // ---- the messages of all CTAs, one a lane (lanes from cs on: none)
  auto exchange = [&](const Message& m) {  // m: thread 0's
    if (tid == 0) box[parity] = m;
    sync_cluster();
    Message got{NEG_INF, kNone, 0.0};
    if (lane < static_cast<int>(cs)) {
      const uint32_t at = mapa_u32(smem_u32(&box[parity]), lane);
      uint32_t w0, w1, w2, w3;
      asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w0), "=r"(w1), "=r"(w2), "=r"(w3)
                   : "r"(at)
                   : "memory");
      got.top = __uint_as_float(w0);
      got.first = static_cast<int>(w1);
      got.sum = __hiloint2double(static_cast<int>(w3), static_cast<int>(w2));
    }
    parity ^= 1;  // (the next exchange's barrier comes before this box is written again)
    return got;
  };
  auto max_of = [](float v) {  // over the warp (no NaN), by an integer of the same order
    const uint32_t u = __float_as_uint(v + 0.f);
    const uint32_t k = __reduce_max_sync(0xffffffffu, (u >> 31) ? ~u : u | 0x80000000u);
    return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
  };
  auto scale_to = [&](float from, float to) { return from == to ? 1.f : ex2((from - to) * c); };
  auto sum_lanes = [&](double v) {
    for (int o = 1; o < kMaxCluster; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return __shfl_sync(0xffffffffu, v, 0);
  };

  // ---- a node's row: its maximum and sum with fp32 weights
  auto read_row = [&](bool odd) {
    float m = NEG_INF, s = 0.f;
    int at = kNone;
    auto take = [&](float mv, int i) {  // a new maximum of this lane
      s *= m == NEG_INF ? 0.f : ex2((m - mv) * c);
      m = mv, at = i;
    };
    if (!odd) {
      // four instructions an element: NaN logits, or infinities at the top, leave a NaN in the sum (and the
      // row is read again)
      auto single = [&](int x) {
        const float l = R::one(row + x);
        if (l > m || at == kNone) take(l, x);
        s += greedy ? (l == l ? 0.f : l) : ex2(fmaf(l, c, m == NEG_INF ? 0.f : -m * c));
      };
      if (lane < head) single(lane);
      const int v0 = vec0();
      const uint4* vec = reinterpret_cast<const uint4*>(row + v0);
      constexpr int U = 5;  // loads in flight
      for (int i0 = lo + lane; i0 < hi; i0 += 32 * U) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (i0 + u * 32 < hi) v[u] = vec[i0 + u * 32];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (i0 + u * 32 >= hi) break;
          float x[8], mv;
          R::many(v[u], x);
          mv = max3(x[0], x[1], x[2]);
#pragma unroll
          for (int e = 3; e < N; e += 2) mv = max3(mv, x[e], x[e + 1 < N ? e + 1 : e]);
          if (mv != mv) s = mv;
          if (mv > m || at == kNone) {
            int e0 = 0;
#pragma unroll
            for (int e = N - 1; e >= 0; --e)
              if (x[e] == mv) e0 = e;
            take(mv, v0 + (i0 + u * 32) * N + e0);
          }
          if (!greedy) {
            const float mc = m == NEG_INF ? 0.f : m * c;
            float add = 0.f, add2 = 0.f;
#pragma unroll
            for (int e = 0; e < N; e += 2) add += ex2(fmaf(x[e], c, -mc)), add2 += ex2(fmaf(x[e + 1], c, -mc));
            s += add + add2;
          }
        }
      }
      if (lane < tail) single(V - tail + lane);
    } else {
      bool nan = false;
      int from, to;
      range(rank * kWarps + warp, from, to);
#pragma unroll 1
      for (int x = from + lane; x < to; x += 32) {
        float l = R::one(row + x);
        nan |= l != l;
        l = clean(l);
        if (l > m || at == kNone) take(l, x);
        if (!greedy) s += l == m ? 1.f : ex2((l - m) * c);
      }
      if (nan) set_err(a.err, kErrNanScore);
    }
    if (at == kNone) s = 0.f;
    const float wm = max_of(m);
    const int wa = static_cast<int>(__reduce_min_sync(0xffffffffu, static_cast<uint32_t>(m == wm ? at : kNone)));
    s *= scale_to(m, wm);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __syncthreads();  // the previous node's sums have been read
    if (lane == 0) w_top[warp] = wm, w_first[warp] = wa, w_sum[warp] = static_cast<double>(s);
    __syncthreads();
    // the CTA's, in every warp: lanes are its warps
    const float own_top = lane < kWarps ? w_top[lane] : NEG_INF;
    const double own_sum = lane < kWarps ? w_sum[lane] : 0.0;
    const float cm = max_of(own_top);
    const int ca = static_cast<int>(
        __reduce_min_sync(0xffffffffu, static_cast<uint32_t>(lane < kWarps && own_top == cm ? w_first[lane] : kNone)));
    double sum = own_sum * static_cast<double>(scale_to(own_top, cm));
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const Message got = exchange(Message{cm, ca, sum});
    top = max_of(got.top);
    eps = base_eps + 0x1.8p-23f * fabsf(top * c);  // (c times the maximum is rounded before the difference)
    first = static_cast<int>(__reduce_min_sync(0xffffffffu, static_cast<uint32_t>(got.top == top ? got.first : kNone)));
    S = sum_lanes(got.sum * static_cast<double>(scale_to(got.top, top)));
    if (warp == 0 && lane < kWarps) w_sum[lane] = own_sum * static_cast<double>(scale_to(own_top, top));
  };
  // ---- a warp's share ``v`` of the sum of what ``n`` rejections leave, to s_R[n] (and each warp's to w_sum)
  auto join_sum = [&](int n, double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) w_sum[warp] = v;
    __syncthreads();
    double sum = lane < kWarps ? w_sum[lane] : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const Message got = exchange(Message{0.f, 0, sum});
    const double all = sum_lanes(got.sum);
    if (tid == 0) s_R[n] = all, s_inv[n] = 1.0 / all, s_finv[n] = static_cast<float>(1.0 / all);
    __syncthreads();
  };
  auto sum_exact = [&](int n) {  // in double
    const int keep = n_rej;
    n_rej = n;
    double v = 0.0;
    int from, to;
    range(rank * kWarps + warp, from, to);
    constexpr int U = 4;
    for (int x = from + lane; x < to; x += 32 * U) {
      float l[U], qx[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool in = x + u * 32 < to;
        l[u] = in ? clean(R::one(row + x + u * 32)) : NEG_INF;
        qx[u] = in && drawn && n ? q[x + u * 32] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (x + u * 32 < to) v += rest_of(x + u * 32, l[u], qx[u]);
    }
    n_rej = keep;
    join_sum(n, v);
  };
  auto sum_fast = [&](int n) {  // (a random draft) in fp32; E from n - 1 to n
    float v = 0.f;
    const int v0 = vec0();
    const uint4* vec = reinterpret_cast<const uint4*>(row + v0);
    const float* qv = q + v0;
    const bool whole = (reinterpret_cast<uintptr_t>(qv) & 15) == 0;
    const float tc = top * c;
    // (a NaN logit gives 0: its product is no larger than 0)
    auto pass = [&](auto left) {
      if (lane < head) v += left(R::one(row + lane), q[lane]);
      constexpr int U = 2;
      for (int i0 = lo + lane; i0 < hi; i0 += 32 * U) {
        uint4 t[U];
        float4 d[U][N / 4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + u * 32;
          if (i >= hi) break;
          t[u] = vec[i];
#pragma unroll
          for (int k = 0; k < N / 4; ++k) {
            const float* at = qv + static_cast<size_t>(i) * N + k * 4;
            d[u][k] = whole ? *reinterpret_cast<const float4*>(at) : make_float4(at[0], at[1], at[2], at[3]);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (i0 + u * 32 >= hi) break;
          float x[8], add = 0.f;
          R::many(t[u], x);
#pragma unroll
          for (int k = 0; k < N / 4; ++k) {
            add += left(x[4 * k], d[u][k].x) + left(x[4 * k + 1], d[u][k].y);
            add += left(x[4 * k + 2], d[u][k].z) + left(x[4 * k + 3], d[u][k].w);
          }
          v += add;
        }
      }
      if (lane < tail) v += left(R::one(row + V - tail + lane), q[V - tail + lane]);
    };
    const float f0 = s_finv[0], f1 = s_finv[1];
    if (n == 1)
      pass([&](float l, float qx) { return fmaxf(fmaf(ex2(fmaf(l, c, -tc)), f0, -qx), 0.f); });
    else
      pass([&](float l, float qx) {
        float r = fmaxf(fmaf(ex2(fmaf(l, c, -tc)), f0, -qx), 0.f);
        r = fmaxf(fmaf(r, f1, -qx), 0.f);
        for (int j = 2; j < n; ++j) r = fmaxf(fmaf(r, s_finv[j], -qx), 0.f);
        return r;
      });
    // weights off by E in all (at first by eps of their sum), divided by a sum that is as far off
    E = (n == 1 ? 2.0 * eps : (2.0 * E + sum_eps * s_R[n - 1]) * s_inv[n - 1]) + 0x1p-22;
    join_sum(n, static_cast<double>(v));
  };
  auto make_exact = [&]() {  // every sum of the current node again, in double
    exact = true;
    for (int k = drawn ? 0 : n_rej; k <= n_rej; ++k) sum_exact(k);
  };

  auto enter = [&](int node) {
    row = reinterpret_cast<const L*>(a.target) + (static_cast<long long>(b) * T + node) * a.ldt;
    if (drawn) q = a.draft + (static_cast<long long>(b) * T + node) * a.ldd;
    n_rej = 0;
    exact = false;
    share();
    read_row(false);
    // A bound that is no small number bounds nothing (its terms are first order): at very low temperatures, c times
    // a logit is rounded by more than the differences that count.  (It is infinite where the maximum is.)
    odd_row = !(S >= 0.0) || !(eps < 0x1p-4f);
    if (odd_row) {
      read_row(true);
      if (tid == 0 && rank == 0 && top == NEG_INF) set_err(a.err, kErrNanScore);  // (all the same weight then)
      // a bound that decides nothing sends tests and draws to the double sums (a sum that is none: as at an
      // infinite temperature)
      if (!(eps < 0x1p-4f && S > 0.5 && S < 4.0 * V)) eps = 1e30f, S = 1.0;
    }
    if (tid == 0) s_R[0] = greedy ? 1.0 : S, s_inv[0] = 1.0 / S, s_finv[0] = static_cast<float>(1.0 / S);
    E = 0.0;
    __syncthreads();
  };

  enter(0);
  int cur = 0, n = 1;
  if (rank == 0 && tid == 0) path[0] = 0;
  for (int j = 1; j < T; ++j) {
    if (s_par[j] != cur) continue;
    const int x = s_tok[j];
    if (x < 0 || x >= V) {
      if (rank == 0 && tid == 0) set_err(a.err, kErrIndex);
      continue;
    }
    const double lhs = static_cast<double>(s_u[j]) *
                       (drawn ? static_cast<double>(q[x]) : 1.0);
    const double rx = rest(x, clean(R::one(row + x)));
    bool yes;
    if (exact || greedy) {
      yes = lhs * s_R[n_rej] < rx;
    } else {
      const double left = s_R[n_rej];
      const double off = drawn && n_rej ? E + sum_eps * left : S * eps;
      yes = lhs * (left + off) < rx - E;
      if (!yes && lhs * (left - off) < rx + E) {  // too near to say
        make_exact();
        yes = lhs * s_R[n_rej] < rest(x, clean(R::one(row + x)));
      }
    }
    if (yes) {
      if (rank == 0 && tid == 0) path[n] = j;
      ++n;
      cur = j;
      enter(j);
      continue;
    }
    if (drawn) {
      ++n_rej;
      if (exact)
        sum_exact(n_rej);
      else if (odd_row)
        make_exact();
      else {
        sum_fast(n_rej);
        if (!(E < 0.25 * s_R[n_rej])) make_exact();  // nothing to go by
      }
    } else {
      __syncthreads();  // s_R[n_rej] has been read
      if (tid == 0) {
        s_rej[n_rej] = x;
        s_R[n_rej + 1] = s_R[n_rej] - rx;
      }
      ++n_rej;
      __syncthreads();
      if (exact && !greedy) sum_exact(n_rej);
    }
  }
  if (rank == 0) {
    for (int i = n + tid; i < T; i += kThreads) path[i] = -1;
    for (int i = tid; i < T; i += kThreads)
      if (s_par[i] >= i) set_err(a.err, kErrIndex);  // names no earlier node: matched no accepted one
    if (tid == 0) a.n_path[b] = n;
  }
  // ---- the next token
  if (greedy) {
    if (rank == 0 && tid == 0) a.next_token[b] = first;
    sync_cluster();  // messages are read before a CTA leaves
    return;
  }
  for (int round = 0;; ++round) {
    // sums of the warps before this one: the CTAs', then the warps'
    double mine = lane < kWarps ? w_sum[lane] : 0.0;
    if (!exact && !drawn && lane < kWarps && n_rej) {  // rejected tokens leave their warps' fp32 sums
      int from, to;
      range(rank * kWarps + lane, from, to);
      for (int j = 0; j < n_rej; ++j) {
        const int x = s_rej[j];
        bool again = false;
        for (int k = 0; k < j; ++k) again |= s_rej[k] == x;
        if (x >= from && x < to && !again) mine -= weight(clean(R::one(row + x)));
      }
    }
    double incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    const double cta = __shfl_sync(0xffffffffu, incl, 31);
    const Message got = exchange(Message{0.f, 0, cta});
    double upto = got.sum;
#pragma unroll
    for (int o = 1; o < kMaxCluster; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    const double total = __shfl_sync(0xffffffffu, upto, kMaxCluster - 1);
    if (exact && !(total > 0.0) && n_rej) {  // nothing is left: the node's own distribution
      n_rej = 0;
      sum_exact(0);
      continue;
    }
    const double want = static_cast<double>(draw) * total;
    // the CTA and the warp where the sum passes the border (or the last ones with any weight)
    const uint32_t over = __ballot_sync(0xffffffffu, lane < static_cast<int>(cs) && got.sum > 0.0 && upto > want);
    const uint32_t some = __ballot_sync(0xffffffffu, lane < static_cast<int>(cs) && got.sum > 0.0);
    const int owner = over ? __ffs(over) - 1 : some ? 31 - __clz(some) : 0;
    const double before = __shfl_sync(0xffffffffu, upto - got.sum, owner);
    if (static_cast<int>(rank) == owner) {
      const uint32_t wo = __ballot_sync(0xffffffffu, lane < kWarps && mine > 0.0 && before + incl > want);
      const uint32_t ws = __ballot_sync(0xffffffffu, lane < kWarps && mine > 0.0);
      const int w = wo ? __ffs(wo) - 1 : ws ? 31 - __clz(ws) : 0;
      double sum = before + __shfl_sync(0xffffffffu, incl - mine, w);
      // that warp's share again, split over the CTA's warps: their sums, then the one that has the border
      int from, to;
      range(rank * kWarps + w, from, to);
      const int count = to - from;
      to = from + static_cast<int>(static_cast<long long>(count) * (warp + 1) / kWarps);
      from += static_cast<int>(static_cast<long long>(count) * warp / kWarps);
      auto value = [&](int x) {
        const float l = clean(R::one(row + x));
        return exact ? rest(x, l) : static_cast<double>(rest_fast(x, l));
      };
      double part = 0.0;
#pragma unroll 1
      for (int x = from + lane; x < to; x += 32) part += value(x);
#pragma unroll
      for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      if (lane == 0) s_part[warp] = part;
      __syncthreads();
      const double parts = lane < kWarps ? s_part[lane] : 0.0;
      double pin = parts;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, pin, o);
        if (lane >= o) pin += t;
      }
      const uint32_t po = __ballot_sync(0xffffffffu, lane < kWarps && parts > 0.0 && sum + pin > want);
      const uint32_t ps = __ballot_sync(0xffffffffu, lane < kWarps && parts > 0.0);
      const int sub = po ? __ffs(po) - 1 : ps ? 31 - __clz(ps) : 0;
      sum += __shfl_sync(0xffffffffu, pin - parts, sub);
      if (warp == sub) {
        int pick = kNone, any = -1;
        bool sure = exact;
        const double off = exact ? 0.0 : drawn && n_rej ? 2.0 * (E + sum_eps * total) : 2.0 * S * eps;
#pragma unroll 1
        for (int x0 = from; x0 < to && pick == kNone; x0 += 32) {
          const int x = x0 + lane;
          const double r = x < to ? value(x) : 0.0;
          double inc = r;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
          }
          const bool over_here = r > 0.0 && sum + inc > want;
          const uint32_t hit = __ballot_sync(0xffffffffu, over_here);
          const uint32_t has = __ballot_sync(0xffffffffu, r > 0.0);
          if (hit) {
            const int l0 = __ffs(hit) - 1;
            pick = x0 + l0;
            // the border lies inside the token's own stretch by more than the sums are off
            sure = exact || __shfl_sync(0xffffffffu, sum + inc - r + off <= want && sum + inc - off > want, l0);
          }
          if (has) any = x0 + 31 - __clz(has);
          sum += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (lane == 0) {
          s_token[0] = pick != kNone ? pick : any;
          s_token[1] = sure || (exact && pick == kNone);
        }
      }
    }
    sync_cluster();
    uint32_t token, certain;
    const uint32_t from = mapa_u32(smem_u32(s_token), owner);
    asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(token), "=r"(certain) : "r"(from) : "memory");
    if (certain) {
      if (rank == 0 && tid == 0) a.next_token[b] = static_cast<int>(token);
      break;
    }
    sync_cluster();  // the token is read before it is made again
    make_exact();
  }
  sync_cluster();  // messages are read before a CTA leaves
}

}  // namespace tv
}  // namespace kvbp

#include "../../include/kvbp.h"

extern "C" int64_t kvbp_tree_verify_workspace(int32_t B, int32_t T, int32_t vocab) {
  (void)B, (void)T, (void)vocab;
  return 0;
}

extern "C" int kvbp_tree_verify(kvbp_stream_t stream, int32_t B, int32_t T, int32_t vocab, int32_t fp32_target,
                                const void* target, int64_t ldt, const float* temperature, const int32_t* tokens,
                                const int32_t* parents, const float* draft_probs, int64_t ldd, const float* accept_u,
                                const float* sample_u, int32_t* path, int32_t* n_path, int32_t* next_token,
                                void* workspace, int64_t workspace_bytes, int32_t* dev_err) {
  using namespace kvbp;
  (void)workspace, (void)workspace_bytes;
  if (!target || !tokens || !parents || !accept_u || !sample_u || !path || !n_path || !next_token)
    return fail(kStatusArg, "tree_verify: null pointer");
  if (B <= 0 || vocab <= 0 || B > 1 << 24 || vocab > 0x7fffffff - 1024) return fail(kStatusArg, "tree_verify: bad size");
  if (T <= 0 || T > tv::kMaxNodes) return fail(kStatusUnsupported, "tree_verify: %d nodes (1 to %d)", T, tv::kMaxNodes);
  if (ldt < vocab || (draft_probs && ldd < vocab)) return fail(kStatusArg, "tree_verify: rows overlap");
  if (misaligned(target, fp32_target ? 4 : 2) || misaligned(draft_probs, 4))
    return fail(kStatusArg, "tree_verify: misaligned rows");
  tv::Args a{T, vocab, target, ldt, temperature, tokens, parents, draft_probs, ldd, accept_u, sample_u, path, n_path,
             next_token, dev_err};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // CTAs of a sequence: as many as a portable cluster has, for what takes the time is the longest path's chain
  // of rows (64 sequences with a draft: 260 us with clusters of 4, 230 with 8); fewer from 75 sequences on,
  // where the rows' bytes do.  CTAs of 512 threads while all are resident, one an SM; else of 256, two an SM
  // (24 sequences: 47 us with 512, 30 with 256; one sequence with a draft: 46 and 54).
  int cs = 8;
  while (cs > 1 && static_cast<long long>(B) * cs > 4 * 148) cs /= 2;
  const bool wide = static_cast<long long>(B) * cs <= 120;  // (clusters of 8 that fit: 15)
  auto kernel = fp32_target ? (wide ? tv::verify_kernel<float, 512> : tv::verify_kernel<float, 256>)
                            : (wide ? tv::verify_kernel<__nv_bfloat16, 512> : tv::verify_kernel<__nv_bfloat16, 256>);
  cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(B) * cs), dim3(wide ? 512 : 256), 0, st, dim3(cs, 1, 1), a);
  if (e != cudaSuccess) return fail(kStatusCuda, "tree_verify launch: %s", cudaGetErrorString(e));
  return kStatusOk;
}
