// Matrix product in 8-bit integers with a scale for each token and each output channel:
//   y[m][n] = (sum_k xq[m][k] wq[n][k]) * sx[m] * sw[n] (+ bias[n])
// with exact 32-bit integer sums, and the per-token quantisation that feeds it.
#include "common.cuh"
#include "kvbp_internal.h"

namespace kvbp {
namespace i8 {

// Per-token quantisation: sx = max|x| / 127, xq = rint(127 x / max|x|) (127 x is exact in
// fp32, so half-way values are half-way in any precision; a zero row gives zeros and scale
// 0).  A row with a NaN or an infinity gets a scale that is not finite, and codes 0: every
// output of that token is then NaN.  One CTA per row, the row kept in registers between the
// maximum and the codes (kVec 16-byte vectors per thread cover K <= 16384; longer rows are
// read again, from L2).
constexpr int kVec = 8;
__global__ void __launch_bounds__(256) quant_rows_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, int K,
                                                         int vec, int8_t* __restrict__ q, long long ldq,
                                                         float* __restrict__ scale) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ uint32_t red[8];
  const size_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const __nv_bfloat16* row = x + r * ldx;
  int8_t* dst = q + r * ldq;
  const int nv = vec ? K / 8 : 0;
  const uint4* rv = reinterpret_cast<const uint4*>(row);
  uint4 keep[kVec];
  uint32_t m = 0;  // max|x| as bits: a NaN's bits are the largest
  auto fold = [&](const uint4 w) {
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) m = max(m, max((ws[k] << 16) & 0x7fffffffu, ws[k] & 0x7fff0000u));
  };
#pragma unroll
  for (int u = 0; u < kVec; ++u) {
    const int i = tid + 256 * u;
    keep[u] = i < nv ? rv[i] : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int u = 0; u < kVec; ++u) fold(keep[u]);
  for (int i = tid + 256 * kVec; i < nv; i += 256) fold(rv[i]);
  for (int i = nv * 8 + tid; i < K; i += 256) m = max(m, __float_as_uint(__bfloat162float(row[i])) & 0x7fffffffu);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((tid & 31) == 0) red[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = max(m, red[w]);
  const float top = __uint_as_float(m);
  const bool fine = m > 0 && m < 0x7f800000u;
  if (tid == 0) scale[r] = top / 127.0f;
  auto code = [&](float v) -> uint32_t {
    return fine ? static_cast<uint32_t>(static_cast<int>(rintf(127.0f * v / top))) & 255u : 0u;
  };
  auto emit = [&](const uint4 w, int i) {
    *reinterpret_cast<uint2*>(dst + 8 * i) = make_uint2(
        code(bf16lo(w.x)) | code(bf16hi(w.x)) << 8 | code(bf16lo(w.y)) << 16 | code(bf16hi(w.y)) << 24,
        code(bf16lo(w.z)) | code(bf16hi(w.z)) << 8 | code(bf16lo(w.w)) << 16 | code(bf16hi(w.w)) << 24);
  };
#pragma unroll
  for (int u = 0; u < kVec; ++u) {
    const int i = tid + 256 * u;
    if (i < nv) emit(keep[u], i);
  }
  for (int i = tid + 256 * kVec; i < nv; i += 256) emit(rv[i], i);
  for (int i = nv * 8 + tid; i < K; i += 256) dst[i] = static_cast<int8_t>(code(__bfloat162float(row[i])));
}

struct Args {
  const int8_t* w;
  long long ldw;
  const float* sw;
  const int8_t* xq;
  long long ldq;
  const float* sx;
  const __nv_bfloat16* bias;
  void* out;
  long long ldo;
  int M, N, K, f32;
};

__device__ __forceinline__ void store(const Args& a, int m, int n, int acc, float sx, float sw, float bias) {
  const float y = static_cast<float>(acc) * sx * sw + bias;
  const size_t at = static_cast<size_t>(m) * a.ldo + n;
  if (a.f32)
    static_cast<float*>(a.out)[at] = y;
  else
    static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
}

// 64 x 64 output tile per CTA, 64-byte K steps in shared memory, dp4a.
__global__ void __launch_bounds__(256) gemm_kernel(const Args a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ int sx[64][17], sw[64][17];
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tid = threadIdx.x;
  const int tm = tid / 16, tn = tid % 16;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < a.K; k0 += 64) {
    for (int i = tid; i < 64 * 16; i += 256) {
      const int r = i / 16, k = k0 + (i % 16) * 4;
      uint32_t vx = 0, vw = 0;
      for (int e = 0; e < 4; ++e) {
        if (k + e < a.K && m0 + r < a.M) vx |= static_cast<uint32_t>(static_cast<uint8_t>(a.xq[static_cast<size_t>(m0 + r) * a.ldq + k + e])) << (8 * e);
        if (k + e < a.K && n0 + r < a.N) vw |= static_cast<uint32_t>(static_cast<uint8_t>(a.w[static_cast<size_t>(n0 + r) * a.ldw + k + e])) << (8 * e);
      }
      sx[r][i % 16] = static_cast<int>(vx);
      sw[r][i % 16] = static_cast<int>(vw);
    }
    __syncthreads();
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(sx[tm + 16 * i][k], sw[tn + 16 * j][k], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + tm + 16 * i, n = n0 + tn + 16 * j;
      if (m < a.M && n < a.N)
        store(a, m, n, acc[i][j], a.sx[m], a.sw[n], a.bias ? __bfloat162float(a.bias[n]) : 0.f);
    }
}

static bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

static int quant_rows(cudaStream_t st, int rows, int K, const void* x, long long ldx, void* q, long long ldq, float* scale) {
  if (!x || !q || !scale) return fail(kStatusArg, "int8_quant_rows: null pointer");
  if (rows <= 0 || K <= 0 || ldx < K || ldq < K) return fail(kStatusArg, "int8_quant_rows: bad size");
  if (misaligned(q, 16) || ldq % 16) return fail(kStatusArg, "int8_quant_rows: q rows must be 16-byte aligned");
  // 16-byte loads where x's rows allow them, else one value at a time
  const int vec = !misaligned(x, 16) && ldx % 8 == 0;
  const cudaError_t e = launch_pdl(quant_rows_kernel, dim3(rows), dim3(256), 0, st, dim3(0),
                                   static_cast<const __nv_bfloat16*>(x), ldx, K, vec, static_cast<int8_t*>(q), ldq, scale);
  if (e != cudaSuccess) return fail(kStatusCuda, "int8_quant_rows launch: %s", cudaGetErrorString(e));
  return kStatusOk;
}

static int gemm(cudaStream_t st, const Args& a) {
  if (!a.w || !a.sw || !a.xq || !a.sx || !a.out) return fail(kStatusArg, "int8_gemm: null pointer");
  if (a.M <= 0 || a.N <= 0 || a.K <= 0 || a.ldw < a.K || a.ldq < a.K || a.ldo < a.N) return fail(kStatusArg, "int8_gemm: bad size");
  // the sum of K products of up to 127 * 127 (128 * 128 for raw codes) stays in 32 bits
  if (a.K > 131071) return fail(kStatusUnsupported, "int8_gemm: K %d > 131071 could overflow the 32-bit sums", a.K);
  if (misaligned(a.w, 16) || misaligned(a.xq, 16) || a.ldw % 16 || a.ldq % 16)
    return fail(kStatusArg, "int8_gemm: w and xq rows must be 16-byte aligned");
  const cudaError_t e = launch_pdl(gemm_kernel, dim3((a.N + 63) / 64, (a.M + 63) / 64), dim3(256), 0, st, dim3(0), a);
  if (e != cudaSuccess) return fail(kStatusCuda, "int8_gemm launch: %s", cudaGetErrorString(e));
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
  (void)dev_err;
  kvbp::i8::Args a{static_cast<const int8_t*>(w), ldw, w_scale, static_cast<const int8_t*>(xq), ldq, x_scale,
                   static_cast<const __nv_bfloat16*>(bias), out, ldo, M, N, K, fp32_out ? 1 : 0};
  return kvbp::i8::gemm(reinterpret_cast<cudaStream_t>(stream), a);
}
