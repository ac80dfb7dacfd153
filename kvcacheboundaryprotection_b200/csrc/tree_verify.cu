// Verification of drafted tokens against the target's probabilities (speculative decoding).
//
// One walk over a sequence's nodes j = 1 .. T-1 in order: a node whose parent is the last
// accepted node is tested.  With r the target's weights at that parent (what earlier siblings
// left of them), R their sum, x the node's token and q the distribution that x was drawn from
// (1 at x where there is none), the node is accepted when u * q(x) * R < r(x); otherwise
//   r <- max(r / R - q, 0)        (r(x) <- 0 where q is 1 at x).
// Each test keeps the target's law: P(accept x) + the residual's mass add up to r / R.  The
// last accepted node's r gives one more token: the first x whose running sum exceeds u * R.
//
// Weights and sums are double: a token is chosen where a running sum of a hundred thousand
// terms passes a border, and 32 bits would choose another one every few hundred draws.
#include <math.h>

#include "common.cuh"
#include "kvbp_internal.h"

namespace kvbp {
namespace tv {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxNodes = 128;

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

__device__ __forceinline__ float logit(const float* row, int x) { return row[x]; }
__device__ __forceinline__ float logit(const __nv_bfloat16* row, int x) { return __bfloat162float(row[x]); }

template <typename L>
__global__ void __launch_bounds__(kThreads) verify_kernel(Args a) {
  __shared__ float red_f[kWarps];
  __shared__ int red_i[kWarps];
  __shared__ double red_d[kWarps];
  __shared__ double s_R[kMaxNodes + 1];
  __shared__ int s_rej[kMaxNodes];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int T = a.T, V = a.V;
  const float NEG_INF = -__int_as_float(0x7f800000);
  const int* par = a.parents + static_cast<size_t>(b) * T;
  const int* tok = a.tokens + static_cast<size_t>(b) * T;
  int* path = a.path + static_cast<size_t>(b) * T;
  const float heat = a.temperature ? a.temperature[b] : 1.f;
  const bool greedy = !(heat > 0.f);
  const double inv = 1.0 / static_cast<double>(greedy ? 1.f : heat);
  if (par[0] != -1) {  // no tree
    for (int i = tid; i < T; i += kThreads) path[i] = -1;
    if (tid == 0) {
      a.n_path[b] = 0;
      a.next_token[b] = -1;
    }
    return;
  }
  const bool drawn = a.draft && !greedy;
  const L* row = nullptr;
  const float* q = nullptr;
  float top = 0.f;
  int first = 0, n_rej = 0;
  // weight of token x at the current node before any rejection
  auto weight = [&](int x) -> double {
    if (greedy) return x == first ? 1.0 : 0.0;
    const float l = logit(row, x);
    if (l == top) return 1.0;
    return l < top ? exp((static_cast<double>(l) - static_cast<double>(top)) * inv) : 0.0;  // NaN: none
  };
  auto rest = [&](int x) -> double {  // what the rejections left of it
    double r = weight(x);
    for (int j = 0; j < n_rej; ++j) {
      if (drawn)
        r = fmax(r / s_R[j] - static_cast<double>(q[x]), 0.0);
      else if (x == s_rej[j])
        r = 0.0;
    }
    return r;
  };
  auto block_sum = [&](double v) -> double {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) red_d[warp] = v;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < kWarps; ++w) t += red_d[w];
    return t;
  };
  auto enter = [&](int node) {  // statistics of a node's row
    row = reinterpret_cast<const L*>(a.target) + (static_cast<long long>(b) * T + node) * a.ldt;
    if (drawn) q = a.draft + (static_cast<long long>(b) * T + node) * a.ldd;
    float m = NEG_INF;
    int at = 0x7fffffff;
    bool nan = false;
    for (int x = tid; x < V; x += kThreads) {
      const float l = logit(row, x);
      nan |= l != l;
      if (l > m || (l == m && x < at)) {
        m = l;
        at = x;
      }
    }
    if (nan) set_err(a.err, kErrNanScore);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
      const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
      if (m2 > m || (m2 == m && a2 < at)) {
        m = m2;
        at = a2;
      }
    }
    __syncthreads();
    if (lane == 0) {
      red_f[warp] = m;
      red_i[warp] = at;
    }
    __syncthreads();
    top = red_f[0];
    first = red_i[0];
    for (int w = 1; w < kWarps; ++w)
      if (red_f[w] > top || (red_f[w] == top && red_i[w] < first)) {
        top = red_f[w];
        first = red_i[w];
      }
    n_rej = 0;
    double sum = 0.0;
    if (!greedy)
      for (int x = tid; x < V; x += kThreads) sum += weight(x);
    sum = block_sum(sum);
    if (tid == 0) s_R[0] = greedy ? 1.0 : sum;
    __syncthreads();
  };

  enter(0);
  int cur = 0, n = 1;
  if (tid == 0) path[0] = 0;
  for (int j = 1; j < T; ++j) {
    if (par[j] != cur) continue;
    const int x = tok[j];
    if (x < 0 || x >= V) {
      if (tid == 0) set_err(a.err, kErrIndex);
      continue;
    }
    const double u = static_cast<double>(a.accept_u[static_cast<size_t>(b) * T + j]);
    const double qx = drawn ? static_cast<double>(q[x]) : 1.0;
    const double rx = rest(x);
    if (u * qx * s_R[n_rej] < rx) {
      if (tid == 0) path[n] = j;
      ++n;
      cur = j;
      __syncthreads();
      enter(j);
      continue;
    }
    // rejected: the sum of what is left
    double left;
    if (drawn) {
      left = 0.0;
      ++n_rej;
      for (int y = tid; y < V; y += kThreads) left += rest(y);
      left = block_sum(left);
    } else {
      left = s_R[n_rej] - rx;
      if (tid == 0) s_rej[n_rej] = x;
      ++n_rej;
      __syncthreads();
    }
    if (tid == 0) s_R[n_rej] = left;
    __syncthreads();
  }
  for (int i = n + tid; i < T; i += kThreads) path[i] = -1;
  // the next token: warps own contiguous ranges, the range where the running sum passes the
  // border is walked again
  const int seg = (V + kWarps - 1) / kWarps;
  const int lo = min(V, warp * seg), hi = min(V, lo + seg);
  auto range_sum = [&]() {
    double v = 0.0;
    for (int x = lo + lane; x < hi; x += 32) v += rest(x);
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  double mine = range_sum(), total = 0.0;
  for (int round = 0; round < 2; ++round) {
    __syncthreads();
    if (lane == 0) red_d[warp] = mine;
    __syncthreads();
    total = 0.0;
    for (int w = 0; w < kWarps; ++w) total += red_d[w];
    if (total > 0.0 || n_rej == 0) break;
    n_rej = 0;  // nothing is left: the node's own distribution
    mine = range_sum();
  }
  const double want = static_cast<double>(a.sample_u[b]) * total;
  double before = 0.0;
  int owner = -1, last = -1;
  double at_owner = 0.0;
  for (int w = 0; w < kWarps; ++w) {
    if (red_d[w] > 0.0) last = w;
    if (owner < 0 && before + red_d[w] > want) {
      owner = w;
      at_owner = before;
    }
    before += red_d[w];
  }
  if (owner < 0) {  // u >= 1, or no weight at all
    owner = last;
    at_owner = before;
  }
  if (owner < 0) {
    if (tid == 0) {
      a.next_token[b] = -1;
      set_err(a.err, kErrNanScore);
    }
  } else if (warp == owner) {
    int pick = 0x7fffffff, any = -1;
    double sum = at_owner;
    for (int x0 = lo; x0 < hi && pick == 0x7fffffff; x0 += 32) {
      const int x = x0 + lane;
      const double r = x < hi ? rest(x) : 0.0;
      double incl = r;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      const uint32_t pos = __ballot_sync(0xffffffffu, r > 0.0);
      const uint32_t over = __ballot_sync(0xffffffffu, r > 0.0 && sum + incl > want);
      if (over) pick = x0 + __ffs(over) - 1;
      if (pos) any = x0 + 31 - __clz(pos);
      sum += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (pick == 0x7fffffff) pick = any;
    if (lane == 0) a.next_token[b] = pick;
  }
  if (tid == 0) a.n_path[b] = n;
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
  if (B <= 0 || vocab <= 0 || B > 65535) return fail(kStatusArg, "tree_verify: bad size");
  if (T <= 0 || T > tv::kMaxNodes) return fail(kStatusUnsupported, "tree_verify: %d nodes (1 to %d)", T, tv::kMaxNodes);
  if (ldt < vocab || (draft_probs && ldd < vocab)) return fail(kStatusArg, "tree_verify: rows overlap");
  if (misaligned(target, fp32_target ? 4 : 2) || misaligned(draft_probs, 4))
    return fail(kStatusArg, "tree_verify: misaligned rows");
  tv::Args a{T, vocab, target, ldt, temperature, tokens, parents, draft_probs, ldd, accept_u, sample_u, path, n_path,
             next_token, dev_err};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (fp32_target)
    tv::verify_kernel<float><<<B, tv::kThreads, 0, st>>>(a);
  else
    tv::verify_kernel<__nv_bfloat16><<<B, tv::kThreads, 0, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(kStatusCuda, "tree_verify launch: %s", cudaGetErrorString(e));
  return kStatusOk;
}
