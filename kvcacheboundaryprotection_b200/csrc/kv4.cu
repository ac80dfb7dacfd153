// Paged KV cache held in 4 bits: append (bias, q/k RMSNorm and RoPE on the way), read-back
// and single-token attention with the per-slot eviction score.
//
// Format.  A pool is [n_pages][Hkv][page_size / 16] blocks of 2304 bytes; a block holds 16
// slots of one kv head.  A row of 128 values is four groups of 32 with one f16 scale each,
//   scale = f16(min(max|x| / 7, 65504)),  code = 8 + clip(rint(x / scale), -7, 7)
// (scale 0: code 8; a NaN in the group: scale NaN).  Symmetric, so that attention needs no
// zero-point sums; f16 scales, so that their rounding (2^-11) is far below half a code step
// and the codes are formed against the rounded scale.
// The block is laid out for the attention kernel's mma.sync fragments (16 x 16 slots x dims
// A operands), so that one 16-byte shared-memory load per thread feeds several MMAs without
// a shuffle or a transpose:
//   0     K codes: slot s at 64 s; dim 32 j + 8 t + n = nibble n of 32-bit word 4 t + j
//   1024  V codes: slot s = 4 t + 2 h + e; dim 32 i + 4 g + n = nibble n of the 16-bit word
//         at 512 h + 64 g + 16 t + 4 i + 2 e (two slots share each 32-bit word: the pair of
//         k columns of the P . V MMA)
//   2048  K scales: slot s, group j at 8 s + 2 j
//   2176  V scales: slot s = 4 t + 2 h + e, group i at 32 t + 16 h + 4 i + 2 e
#include <cuda_fp16.h>

#include "common.cuh"
#include "kvbp_internal.h"

namespace kvbp {
namespace kv4 {

constexpr int kBlock = 2304;  // bytes of 16 slots of one kv head
constexpr int kKScale = 2048;
constexpr int kVScale = 2176;

__device__ __forceinline__ int v_code_offset(int slot, int L) {  // dims 4 L .. 4 L + 3 of slot 0..15
  return 1024 + 512 * ((slot >> 1) & 1) + 64 * (L & 7) + 16 * (slot >> 2) + 4 * (L >> 3) + 2 * (slot & 1);
}
__device__ __forceinline__ int k_code_offset(int slot, int L) {
  return 64 * slot + 16 * ((L & 7) >> 1) + 4 * (L >> 3) + 2 * (L & 1);
}
__device__ __forceinline__ int k_scale_offset(int slot, int j) { return kKScale + 8 * slot + 2 * j; }
__device__ __forceinline__ int v_scale_offset(int slot, int i) {
  return kVScale + 32 * (slot >> 2) + 16 * ((slot >> 1) & 1) + 4 * i + 2 * (slot & 1);
}

// Where slot ``slot`` of sequence ``b`` lives: its block's address for kv head 0 (a head is
// hstride bytes further), or null (with KVBP_DEV_INDEX set) when the slot or its page is
// out of range.  Byte offsets are 64-bit: pools pass 2^31 bytes.
struct Pool {
  uint8_t* base;
  const int* table;
  int B, Hkv, page, n_pages, max_pages;
  __device__ __forceinline__ uint8_t* block_of(int b, int slot, int* err, bool report) const {
    const int pi = slot / page;
    int pg = -1;
    if (b >= 0 && b < B && pi < max_pages) pg = table[static_cast<size_t>(b) * max_pages + pi];
    if (pg < 0 || pg >= n_pages) {
      if (report) set_err(err, kErrIndex);
      return nullptr;
    }
    return base + (static_cast<size_t>(pg) * Hkv * (page / 16) + (slot - pi * page) / 16) * kBlock;
  }
  __device__ __forceinline__ size_t hstride() const { return static_cast<size_t>(page / 16) * kBlock; }
};

// max|x| over the 8 lanes that share a group, as bits: a NaN's bits are the largest, so it
// reaches the scale.
__device__ __forceinline__ uint32_t group_max(uint32_t m) {
#pragma unroll
  for (int o = 4; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
__device__ __forceinline__ __half group_scale(uint32_t amax_bits) {
  if (amax_bits > 0x7f800000u) return __ushort_as_half(0x7fff);
  return __float2half_rn(fminf(__uint_as_float(amax_bits) / 7.0f, 65504.0f));
}
// four codes as one 16-bit word
__device__ __forceinline__ uint32_t four_codes(const float (&x)[4], float scale) {
  uint32_t w = 0;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    // scale 0 (all values below the smallest f16 step) and NaN: code 8, the value 0 * scale
    const float q = scale > 0.f ? fminf(fmaxf(rintf(x[n] / scale), -7.f), 7.f) : 0.f;
    w |= static_cast<uint32_t>(static_cast<int>(q) + 8) << (4 * n);
  }
  return w;
}

// Append.  One CTA per row; half-warp u finishes heads u, u + 16, ... of the row's Hq query,
// Hkv key and Hkv value heads; lane l of the half-warp owns dims 4 l .. 4 l + 3 and
// 64 + 4 l .. 64 + 4 l + 3, so the RoPE pairs (d, d + 64) are its own and a group of 32 dims
// is 8 lanes.  Everything between the bf16 input and the stored value is fp32, rounded once
// (q to bf16, k and v to their codes): the cache keeps 4 bits, so no bf16 step in between
// is worth its error.  The angle pos * inv_freq is reduced in double: at position 4e5 an
// fp32 product would be off by up to 2e-2 rad.
// HBM-bound on a prompt: it reads qkv and writes q once, and 144 bytes per kv head.
__global__ void __launch_bounds__(256) append_kernel(
    const __nv_bfloat16* __restrict__ qkv, int ldq, const __nv_bfloat16* __restrict__ bias,
    const __nv_bfloat16* __restrict__ qnw, const __nv_bfloat16* __restrict__ knw, float eps,
    const float* __restrict__ inv_freq, const int* __restrict__ positions, const int* __restrict__ slots,
    const int* __restrict__ seq, int rows_per_seq, int Hq, Pool pool, __nv_bfloat16* __restrict__ q_out, int* err) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float cs[64], sn[64];
  const int r = blockIdx.x, tid = threadIdx.x, l = tid & 15;
  if (inv_freq) {
    if (tid < 64) {
      const double turns = static_cast<double>(positions[r]) * static_cast<double>(inv_freq[tid]) * 0.15915494309189533577;
      float s, c;
      sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
      cs[tid] = c;
      sn[tid] = s;
    }
    __syncthreads();
  }
  const int slot = slots[r];
  const int b = seq ? seq[r] : r / rows_per_seq;
  uint8_t* blk = slot >= 0 ? pool.block_of(b, slot, err, tid == 0) : nullptr;
  const int in = slot & 15;
  const int nh = Hq + 2 * pool.Hkv;
  // both halves of a warp run the same number of rounds: the shuffles are warp-wide
  for (int h0 = (tid >> 5) * 2; h0 < nh; h0 += 16) {
    const int hh = h0 + ((tid >> 4) & 1);
    const bool live = hh < nh;
    const int hc = live ? hh : nh - 1;
    const __nv_bfloat16* src = qkv + static_cast<size_t>(r) * ldq + hc * 128 + 4 * l;
    const uint2 a = *reinterpret_cast<const uint2*>(src), c = *reinterpret_cast<const uint2*>(src + 64);
    float lo[4] = {bf16lo(a.x), bf16hi(a.x), bf16lo(a.y), bf16hi(a.y)};
    float hi[4] = {bf16lo(c.x), bf16hi(c.x), bf16lo(c.y), bf16hi(c.y)};
    if (bias) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        lo[n] += __bfloat162float(bias[hc * 128 + 4 * l + n]);
        hi[n] += __bfloat162float(bias[hc * 128 + 64 + 4 * l + n]);
      }
    }
    const bool is_q = hc < Hq, is_v = hc >= Hq + pool.Hkv;
    const __nv_bfloat16* nw = is_q ? qnw : knw;
    if (qnw || knw) {
      float ss = 0.f;
#pragma unroll
      for (int n = 0; n < 4; ++n) ss += lo[n] * lo[n] + hi[n] * hi[n];
#pragma unroll
      for (int o = 8; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (!is_v && nw) {
        const float rms = sqrtf(ss / 128.0f + eps);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          lo[n] = lo[n] / rms * __bfloat162float(nw[4 * l + n]);
          hi[n] = hi[n] / rms * __bfloat162float(nw[64 + 4 * l + n]);
        }
      }
    }
    if (inv_freq && !is_v) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float co = cs[4 * l + n], si = sn[4 * l + n];
        const float y = lo[n] * co - hi[n] * si;
        hi[n] = hi[n] * co + lo[n] * si;
        lo[n] = y;
      }
    }
    if (is_q) {
      if (live) {
        __nv_bfloat16* dst = q_out + (static_cast<size_t>(r) * Hq + hc) * 128 + 4 * l;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(lo[0], lo[1]), pack_bf16(lo[2], lo[3]));
        *reinterpret_cast<uint2*>(dst + 64) = make_uint2(pack_bf16(hi[0], hi[1]), pack_bf16(hi[2], hi[3]));
      }
    }
    // every lane of the warp reduces (the other half-warp may hold a key)
    uint32_t ml = 0, mh = 0;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      ml = max(ml, __float_as_uint(fabsf(lo[n])));
      mh = max(mh, __float_as_uint(fabsf(hi[n])));
    }
    ml = group_max(ml);
    mh = group_max(mh);
    if (live && !is_q && blk) {
      uint8_t* dst = blk + static_cast<size_t>(hc - Hq - (is_v ? pool.Hkv : 0)) * pool.hstride();
      const __half sl = group_scale(ml), sh = group_scale(mh);
      const uint32_t wl = four_codes(lo, __half2float(sl)), wh = four_codes(hi, __half2float(sh));
      const int cl = is_v ? v_code_offset(in, l) : k_code_offset(in, l);
      const int ch = is_v ? v_code_offset(in, l + 16) : k_code_offset(in, l + 16);
      *reinterpret_cast<uint16_t*>(dst + cl) = static_cast<uint16_t>(wl);
      *reinterpret_cast<uint16_t*>(dst + ch) = static_cast<uint16_t>(wh);
      if ((l & 7) == 0) {
        const int j = l >> 3;
        *reinterpret_cast<__half*>(dst + (is_v ? v_scale_offset(in, j) : k_scale_offset(in, j))) = sl;
        *reinterpret_cast<__half*>(dst + (is_v ? v_scale_offset(in, j + 2) : k_scale_offset(in, j + 2))) = sh;
      }
    }
  }
}

// Read-back of listed slots as bf16 rows.  One half-warp per (row, kv head).
__global__ void __launch_bounds__(256) gather_kernel(const int* __restrict__ slots, const int* __restrict__ seq,
                                                     int rows_per_seq, long long n, Pool pool,
                                                     __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out,
                                                     long long row_stride, long long head_stride, int* err) {
  pdl_launch_dependents();
  pdl_wait();
  const long long u = static_cast<long long>(blockIdx.x) * 16 + (threadIdx.x >> 4);
  if (u >= n) return;
  const int l = threadIdx.x & 15;
  const long long r = u / pool.Hkv;
  const int h = static_cast<int>(u - r * pool.Hkv);
  const int slot = slots[r];
  const int b = seq ? seq[r] : static_cast<int>(r / rows_per_seq);
  const uint8_t* blk = slot >= 0 ? pool.block_of(b, slot, err, h == 0 && l == 0) : nullptr;
  uint2 o[2][2] = {};
  if (blk) {
    blk += h * pool.hstride();
    const int in = slot & 15;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int L = l + 16 * half, j = L >> 3;
        const uint32_t c = *reinterpret_cast<const uint16_t*>(blk + (w ? v_code_offset(in, L) : k_code_offset(in, L)));
        const float s = __half2float(*reinterpret_cast<const __half*>(blk + (w ? v_scale_offset(in, j) : k_scale_offset(in, j))));
        float x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = static_cast<float>(static_cast<int>((c >> (4 * k)) & 15u) - 8) * s;
        o[w][half] = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
      }
  }
  const long long at = r * row_stride + h * head_stride + 4 * l;
  *reinterpret_cast<uint2*>(k_out + at) = o[0][0];
  *reinterpret_cast<uint2*>(k_out + at + 64) = o[0][1];
  *reinterpret_cast<uint2*>(v_out + at) = o[1][0];
  *reinterpret_cast<uint2*>(v_out + at + 64) = o[1][1];
}

// Attention of one token per sequence.  One CTA of 8 warps per (kv head, sequence); a warp
// takes slots w, w + 8, ... with an online softmax per query head, lane l holding dims
// 4 l .. 4 l + 3; the warps' (max, sum, O) are merged in shared memory.  With a score, a
// second walk over K forms each slot's probabilities from the final (max, sum).
template <int G>
__global__ void __launch_bounds__(256) attend_kernel(const __nv_bfloat16* __restrict__ q, Pool pool,
                                                     const int* __restrict__ lens, const int* __restrict__ slot_pos,
                                                     int S, int limit, float scale, int Hq,
                                                     __nv_bfloat16* __restrict__ out, float* __restrict__ step_score,
                                                     int* err) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float sm[8][G], sl[8][G], so[8][G][128];
  const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = Hq / pool.Hkv;
  int n = lens[b];
  if (n < 0 || n > limit) {
    if (threadIdx.x == 0 && h == 0) set_err(err, kErrIndex);
    n = n < 0 ? 0 : limit;
  }
  float qf[G][4], m[G], l[G], o[G][4];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const uint2 w = g < group ? *reinterpret_cast<const uint2*>(q + (static_cast<size_t>(b) * Hq + h * group + g) * 128 + 4 * lane)
                              : make_uint2(0, 0);
    qf[g][0] = bf16lo(w.x), qf[g][1] = bf16hi(w.x), qf[g][2] = bf16lo(w.y), qf[g][3] = bf16hi(w.y);
    m[g] = -INFINITY, l[g] = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[g][k] = 0.f;
  }
  const float to2 = scale * 1.4426950408889634f;  // logits in units of ln 2
  auto block = [&](int s) -> const uint8_t* {  // the slot's block, null when it is masked
    if (slot_pos && slot_pos[static_cast<size_t>(b) * S + s] < 0) return nullptr;
    const uint8_t* p = pool.block_of(b, s, err, lane == 0 && h == 0);
    return p ? p + h * pool.hstride() : nullptr;
  };
  auto logits = [&](const uint8_t* blk, int in, float (&s)[G]) {
    const uint32_t c = *reinterpret_cast<const uint16_t*>(blk + k_code_offset(in, lane));
    const float ks = __half2float(*reinterpret_cast<const __half*>(blk + k_scale_offset(in, lane >> 3)));
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float d = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) d += qf[g][k] * static_cast<float>(static_cast<int>((c >> (4 * k)) & 15u) - 8);
      d *= ks;
#pragma unroll
      for (int off = 16; off; off >>= 1) d += __shfl_xor_sync(0xffffffffu, d, off);
      s[g] = d * to2;
    }
  };
  bool any = false;
  for (int s = warp; s < n; s += 8) {
    const uint8_t* blk = block(s);
    if (!blk) continue;
    any = true;
    float x[G];
    logits(blk, s & 15, x);
    const uint32_t c = *reinterpret_cast<const uint16_t*>(blk + v_code_offset(s & 15, lane));
    const float vs = __half2float(*reinterpret_cast<const __half*>(blk + v_scale_offset(s & 15, lane >> 3)));
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float mn = fmaxf(m[g], x[g]), f = exp2f(m[g] - mn), p = exp2f(x[g] - mn);
      m[g] = mn;
      l[g] = l[g] * f + p;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        o[g][k] = o[g][k] * f + p * (static_cast<float>(static_cast<int>((c >> (4 * k)) & 15u) - 8) * vs);
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if (lane == 0) sm[warp][g] = m[g], sl[warp][g] = l[g];
#pragma unroll
    for (int k = 0; k < 4; ++k) so[warp][g][4 * lane + k] = o[g][k];
  }
  const int found = __syncthreads_or(any);
  if (!found && n > 0 && threadIdx.x == 0) set_err(err, kErrNoValidSlot);
  float M[G], R[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    M[g] = -INFINITY;
    for (int w = 0; w < 8; ++w) M[g] = fmaxf(M[g], sm[w][g]);
    float L = 0.f;
    for (int w = 0; w < 8; ++w) L += sm[w][g] > -INFINITY ? sl[w][g] * exp2f(sm[w][g] - M[g]) : sl[w][g];
    R[g] = found ? 1.0f / L : 0.f;
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if (g >= group || threadIdx.x >= 128) continue;
    float v = 0.f;
    if (found)
      for (int w = 0; w < 8; ++w) {
        const float f = sm[w][g] > -INFINITY ? exp2f(sm[w][g] - M[g]) : 0.f;
        v += f > 0.f || f != f ? so[w][g][threadIdx.x] * f : 0.f;
      }
    out[(static_cast<size_t>(b) * Hq + h * group + g) * 128 + threadIdx.x] = __float2bfloat16_rn(v * R[g]);
  }
  if (!step_score || !found) return;
  for (int s = warp; s < n; s += 8) {
    const uint8_t* blk = block(s);
    if (!blk) continue;
    float x[G], p = 0.f;
    logits(blk, s & 15, x);
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (g < group) {
        const float e = exp2f(x[g] - M[g]) * R[g];
        if (e != e && lane == 0) set_err(err, kErrNanScore);
        p = fmaxf(p, e);
      }
    if (lane == 0) atomicMax(reinterpret_cast<int*>(step_score + static_cast<size_t>(b) * S + s), __float_as_int(p));
  }
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Checks shared by the three entry points; fills ``p``.
static int make_pool(const char* what, int B, int Hkv, int D, int page, int n_pages, int max_pages, const void* pool,
                     const int* table, Pool* p) {
  if (!pool || !table) return fail(kStatusArg, "%s: null pointer", what);
  if (D != 128) return fail(kStatusUnsupported, "%s: head_dim %d unsupported (only 128)", what, D);
  if (B <= 0 || Hkv <= 0 || n_pages <= 0 || max_pages <= 0) return fail(kStatusArg, "%s: bad size", what);
  if (page <= 0 || page % 16) return fail(kStatusArg, "%s: page_size %d is not a multiple of 16", what, page);
  if (static_cast<long long>(page) * max_pages > 0x7fffffffll - 64)
    return fail(kStatusArg, "%s: %d pages of %d slots exceed 32-bit slot numbers", what, max_pages, page);
  if (!aligned16(pool)) return fail(kStatusArg, "%s: the pool must be 16-byte aligned", what);
  *p = Pool{static_cast<uint8_t*>(const_cast<void*>(pool)), table, B, Hkv, page, n_pages, max_pages};
  return kStatusOk;
}

}  // namespace kv4
}  // namespace kvbp

#include "../../include/kvbp.h"

using kvbp::fail;
namespace kv4 = kvbp::kv4;

extern "C" int kvbp_kv4_append(kvbp_stream_t stream, int32_t rows, int32_t rows_per_seq, const int32_t* seq, int32_t B,
                               int32_t Hq, int32_t Hkv, int32_t head_dim, int32_t page_size, int32_t n_pages,
                               int32_t max_pages, const void* qkv, int32_t ldq, const void* bias, const void* q_norm_w,
                               const void* k_norm_w, float eps, const float* inv_freq, const int32_t* positions,
                               const int32_t* slots, const int32_t* page_table, void* q_out, void* pool,
                               int32_t* dev_err) {
  kv4::Pool p;
  if (int st = kv4::make_pool("kv4_append", B, Hkv, head_dim, page_size, n_pages, max_pages, pool, page_table, &p))
    return st;
  if (!qkv || !slots || (Hq > 0 && !q_out) || (inv_freq && !positions))
    return fail(kvbp::kStatusArg, "kv4_append: null pointer");
  if (rows <= 0 || Hq < 0 || (!seq && rows_per_seq <= 0) || Hq > 65535 || Hkv > 65535 ||
      ldq < (static_cast<long long>(Hq) + 2 * Hkv) * 128)
    return fail(kvbp::kStatusArg, "kv4_append: bad size");
  if (ldq % 4 || ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out)) & 7))
    return fail(kvbp::kStatusArg, "kv4_append: qkv and q_out rows must be 8-byte aligned");
  const cudaError_t e = kvbp::launch_pdl(
      kv4::append_kernel, dim3(rows), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), dim3(0),
      static_cast<const __nv_bfloat16*>(qkv), ldq, static_cast<const __nv_bfloat16*>(bias),
      static_cast<const __nv_bfloat16*>(q_norm_w), static_cast<const __nv_bfloat16*>(k_norm_w), eps, inv_freq,
      positions, slots, seq, rows_per_seq, Hq, p, static_cast<__nv_bfloat16*>(q_out), dev_err);
  if (e != cudaSuccess) return fail(kvbp::kStatusCuda, "kv4_append launch: %s", cudaGetErrorString(e));
  return kvbp::kStatusOk;
}

extern "C" int kvbp_kv4_gather(kvbp_stream_t stream, int32_t rows, int32_t rows_per_seq, const int32_t* seq, int32_t B,
                               int32_t Hkv, int32_t head_dim, int32_t page_size, int32_t n_pages, int32_t max_pages,
                               const int32_t* slots, const int32_t* page_table, const void* pool, void* k_out,
                               void* v_out, int64_t row_stride, int64_t head_stride, int32_t* dev_err) {
  kv4::Pool p;
  if (int st = kv4::make_pool("kv4_gather", B, Hkv, head_dim, page_size, n_pages, max_pages, pool, page_table, &p))
    return st;
  if (!slots || !k_out || !v_out) return fail(kvbp::kStatusArg, "kv4_gather: null pointer");
  if (rows <= 0 || (!seq && rows_per_seq <= 0)) return fail(kvbp::kStatusArg, "kv4_gather: bad size");
  if (row_stride < 128 || head_stride < 128 || row_stride % 4 || head_stride % 4 ||
      ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 7))
    return fail(kvbp::kStatusArg, "kv4_gather: output rows must be 128 apart or more and 8-byte aligned");
  const long long n = static_cast<long long>(rows) * Hkv;
  if ((n + 15) / 16 > 0x7fffffffll) return fail(kvbp::kStatusArg, "kv4_gather: too many rows");
  const cudaError_t e = kvbp::launch_pdl(
      kv4::gather_kernel, dim3(static_cast<unsigned>((n + 15) / 16)), dim3(256), 0,
      reinterpret_cast<cudaStream_t>(stream), dim3(0), slots, seq, rows_per_seq, n, p,
      static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), static_cast<long long>(row_stride),
      static_cast<long long>(head_stride), dev_err);
  if (e != cudaSuccess) return fail(kvbp::kStatusCuda, "kv4_gather launch: %s", cudaGetErrorString(e));
  return kvbp::kStatusOk;
}

extern "C" int64_t kvbp_kv4_attn_workspace(int32_t B, int32_t Hq, int32_t Hkv, int32_t max_slots, int32_t with_score) {
  (void)B, (void)Hq, (void)Hkv, (void)max_slots, (void)with_score;
  return 16;
}

extern "C" int kvbp_kv4_attn(kvbp_stream_t stream, int32_t B, int32_t Hq, int32_t Hkv, int32_t head_dim,
                             int32_t page_size, int32_t n_pages, int32_t max_pages, const void* q, const void* pool,
                             const int32_t* page_table, const int32_t* lens, const int32_t* slot_pos, int32_t S,
                             float scale, void* out, float* step_score, void* workspace, int64_t workspace_bytes,
                             int32_t* dev_err) {
  kv4::Pool p;
  if (int st = kv4::make_pool("kv4_attn", B, Hkv, head_dim, page_size, n_pages, max_pages, pool, page_table, &p))
    return st;
  if (!q || !lens || !out) return fail(kvbp::kStatusArg, "kv4_attn: null pointer");
  if (Hq <= 0 || Hq % Hkv) return fail(kvbp::kStatusArg, "kv4_attn: Hq must be a multiple of Hkv");
  if (Hq / Hkv > 8) return fail(kvbp::kStatusUnsupported, "kv4_attn: query group %d > 8", Hq / Hkv);
  if (S < 0 || ((slot_pos || step_score) && S == 0)) return fail(kvbp::kStatusArg, "kv4_attn: bad slot stride");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15)
    return fail(kvbp::kStatusArg, "kv4_attn: q and out must be 16-byte aligned");
  if (B > 65535 || Hkv > 65535) return fail(kvbp::kStatusArg, "kv4_attn: bad size");
  int limit = max_pages * page_size;
  if ((slot_pos || step_score) && S < limit) limit = S;
  const cudaError_t e = kvbp::launch_pdl(
      kv4::attend_kernel<8>, dim3(Hkv, B), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), dim3(0),
      static_cast<const __nv_bfloat16*>(q), p, lens, slot_pos, S, limit, scale, Hq, static_cast<__nv_bfloat16*>(out),
      step_score, dev_err);
  if (e != cudaSuccess) return fail(kvbp::kStatusCuda, "kv4_attn launch: %s", cudaGetErrorString(e));
  return kvbp::kStatusOk;
}
