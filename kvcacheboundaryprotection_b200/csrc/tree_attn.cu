// Attention of a tree of drafted tokens over the slot cache, with the eviction score of every
// (node, key): out = softmax(scale * q . k) v over the live slots and the node's ancestors.
// One warp per (sequence, node, query head), one pass with the running maximum and sum, a
// second one over the keys where the score is wanted.
#include "common.cuh"
#include "kvbp_internal.h"

namespace kvbp {
namespace ta {

constexpr int kD = 128;
constexpr int kMaxNodes = 128;

struct Args {
  int B, T, Hq, Hkv, S;
  float scale;
  const __nv_bfloat16 *q, *kc, *vc, *kd, *vd;
  const int *parents, *slot_pos, *lens;
  __nv_bfloat16* out;
  float* score;  // [B][T][S + T] or null
  int* err;
};

__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  v[0] = bf16lo(w.x), v[1] = bf16hi(w.x), v[2] = bf16lo(w.y), v[3] = bf16hi(w.y);
}

__global__ void __launch_bounds__(128) simple_kernel(Args a) {
  const int lane = threadIdx.x & 31;
  const int h = blockIdx.x * 4 + (threadIdx.x >> 5), t = blockIdx.y, b = blockIdx.z;
  if (h >= a.Hq) return;
  const int g = h / (a.Hq / a.Hkv);
  const int* par = a.parents + static_cast<size_t>(b) * a.T;
  const size_t row = ((static_cast<size_t>(b) * a.T + t) * a.Hq + h) * kD + lane * 4;
  // the node and its ancestors
  uint32_t sees[kMaxNodes / 32] = {};
  bool used = true;
  for (int j = t, n = 0;; ++n) {
    const int p = par[j];
    sees[j >> 5] |= 1u << (j & 31);
    if (p >= j || p < -1) {
      used = false;
      if (p >= j && lane == 0) set_err(a.err, kErrIndex);
    }
    if (!used || p < 0) break;
    j = p;
  }
  int len = a.lens ? a.lens[b] : a.S;
  if (len < 0 || len > a.S) {
    if (lane == 0) set_err(a.err, kErrIndex);
    len = len < 0 ? 0 : a.S;
  }
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  if (used) {
    float q[4];
    load4(a.q + row, q);
    float m = -__int_as_float(0x7f800000), l = 0.f;
    const size_t head = static_cast<size_t>(b) * a.Hkv + g;
    auto live = [&](int s) {
      return s < a.S ? s < len && (!a.slot_pos || a.slot_pos[static_cast<size_t>(b) * a.S + s] >= 0)
                     : ((sees[(s - a.S) >> 5] >> ((s - a.S) & 31)) & 1u) != 0;
    };
    auto dot = [&](int s) {
      float k[4];
      load4((s < a.S ? a.kc + (head * a.S + s) * kD : a.kd + (head * a.T + (s - a.S)) * kD) + lane * 4, k);
      float d = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
      for (int x = 16; x; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
      return d * a.scale;
    };
    for (int s = 0; s < a.S + a.T; ++s) {
      if (!live(s)) continue;
      const float d = dot(s);
      const float mn = fmaxf(m, d), c = expf(m - mn), p = expf(d - mn);
      float v[4];
      load4((s < a.S ? a.vc + (head * a.S + s) * kD : a.vd + (head * a.T + (s - a.S)) * kD) + lane * 4, v);
      l = l * c + p;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = o[i] * c + p * v[i];
      m = mn;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] /= l;
    if (a.score) {
      float* sc = a.score + (static_cast<size_t>(b) * a.T + t) * (static_cast<size_t>(a.S) + a.T);
      for (int s = 0; s < a.S + a.T; ++s) {
        if (!live(s)) continue;
        const float p = expf(dot(s) - m) / l;
        if (lane == 0) atomicMax(reinterpret_cast<int*>(sc + s), __float_as_int(p));
      }
    }
  }
  *reinterpret_cast<uint2*>(a.out + row) = make_uint2(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]));
}

}  // namespace ta
}  // namespace kvbp

#include "../../include/kvbp.h"

extern "C" int64_t kvbp_tree_attn_workspace(int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t S,
                                            int32_t with_score) {
  (void)B, (void)T, (void)Hq, (void)Hkv, (void)S, (void)with_score;
  return 0;
}

extern "C" int kvbp_tree_attn(kvbp_stream_t stream, int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t head_dim,
                              int32_t S, const void* q, const void* kcache, const void* vcache, const void* k_draft,
                              const void* v_draft, const int32_t* parents, const int32_t* slot_pos,
                              const int32_t* lens, float scale, void* out, float* node_score, void* workspace,
                              int64_t workspace_bytes, int32_t* dev_err) {
  using namespace kvbp;
  (void)workspace, (void)workspace_bytes;
  if (!q || !k_draft || !v_draft || !parents || !out || (S > 0 && (!kcache || !vcache)))
    return fail(kStatusArg, "tree_attn: null pointer");
  if (head_dim != ta::kD) return fail(kStatusUnsupported, "tree_attn: head_dim %d unsupported (only 128)", head_dim);
  if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || S < 0 || B > 65535) return fail(kStatusArg, "tree_attn: bad size");
  if (T <= 0 || T > ta::kMaxNodes) return fail(kStatusUnsupported, "tree_attn: %d nodes (1 to %d)", T, ta::kMaxNodes);
  ta::Args a{B, T, Hq, Hkv, S, scale,
             static_cast<const __nv_bfloat16*>(q), static_cast<const __nv_bfloat16*>(kcache),
             static_cast<const __nv_bfloat16*>(vcache), static_cast<const __nv_bfloat16*>(k_draft),
             static_cast<const __nv_bfloat16*>(v_draft), parents, slot_pos, lens, static_cast<__nv_bfloat16*>(out),
             node_score, dev_err};
  ta::simple_kernel<<<dim3((Hq + 3) / 4, T, B), 128, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(kStatusCuda, "tree_attn launch: %s", cudaGetErrorString(e));
  return kStatusOk;
}
