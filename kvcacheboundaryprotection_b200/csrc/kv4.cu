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

#include <type_traits>

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

// max|x| over the 4 lanes that share a group, as bits: a NaN's bits are the largest, so it
// reaches the scale.
__device__ __forceinline__ uint32_t group_max(uint32_t m) {
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
}
__device__ __forceinline__ __half group_scale(uint32_t amax_bits) {
  if (amax_bits > 0x7f800000u) return __ushort_as_half(0x7fff);
  return __float2half_rn(fminf(__uint_as_float(amax_bits) / 7.0f, 65504.0f));
}
// eight codes as one 32-bit word: clip(rint(x / scale), -7, 7) + 8 each.  x times the rounded
// reciprocal plus 1.5 * 2^23 leaves the integer in the low mantissa bits; only what lies within
// 1e-4 of half-way can round wrongly (bf16 values over an f16 scale often are half-way), and is
// divided.  Scale 0 (all values below the smallest f16 step) and NaN: code 8.
__device__ __forceinline__ uint32_t eight_codes(const float (&x)[8], float scale) {
  const float inv = 1.0f / scale;
  uint32_t w = 0;
  float worst = 0.f;
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const float v = fminf(fmaxf(x[n] * inv, -7.f), 7.f), q = v + (12582912.0f + 8.0f);
    worst = fmaxf(worst, fabsf(v - (q - (12582912.0f + 8.0f))));
    w |= (__float_as_uint(q) & 15u) << (4 * n);
  }
  if (worst > 0.4999f) {
    w = 0;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const float q = fminf(fmaxf(rintf(x[n] / scale), -7.f), 7.f);
      w |= static_cast<uint32_t>(static_cast<int>(q) + 8) << (4 * n);
    }
  }
  return scale > 0.f ? w : 0x88888888u;
}
__device__ __forceinline__ void unpack8(const uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) x[2 * k] = bf16lo(w[k]), x[2 * k + 1] = bf16hi(w[k]);
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
// x[0..7] = p[0..7], one load where all of the call's rows are 16-byte aligned (``wide``)
__device__ __forceinline__ void load8(const __nv_bfloat16* p, bool wide, float (&x)[8]) {
  if (wide) {
    unpack8(*reinterpret_cast<const uint4*>(p), x);
  } else {
#pragma unroll
    for (int n = 0; n < 8; ++n) x[n] = __bfloat162float(p[n]);
  }
}

struct AppendArgs {
  const __nv_bfloat16* qkv;
  const __nv_bfloat16* bias;
  const __nv_bfloat16* qnw;
  const __nv_bfloat16* knw;
  const float* inv_freq;
  const int* positions;
  const int* slots;
  const int* seq;
  Pool pool;
  __nv_bfloat16* q_out;
  int* err;
  int ldq, rows, rows_per_seq, Hq, wide;
  float eps;
};

// Append.  A CTA takes R rows; a warp takes four heads of a row at a time, eight lanes each:
// lane l of the eight owns dims 8 l .. 8 l + 7 and 64 + 8 l .. 64 + 8 l + 7 (16-byte loads),
// so the RoPE pairs (d, d + 64) are its own, a group of 32 dims is four lanes and its eight
// codes are one word of K.  Everything between the bf16 input and the stored value is fp32,
// rounded once (q to bf16, k and v to their codes): the cache keeps 4 bits, so no bf16 step in
// between is worth its error.  Every product, sum and quotient is rounded by itself (no fused
// multiply-add) and the angle pos * inv_freq and its cosine are double: the fp32 values, and so
// the codes of those that sit at a code's border, are the ones that the formula gives step by
// step.  (An fp32 angle would be off by up to 2e-2 rad at position 4e5.)
// Bound by HBM on a prompt (reads qkv, writes q, 144 bytes per kv head): eight rows per CTA
// share one phase of angles, one per thread and half; with few rows one row per CTA spreads
// them over the SMs (latency).
template <int R>
__global__ void __launch_bounds__(256, R > 1 ? 4 : 1) append_kernel(const AppendArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ __align__(16) float cs[R][64], sn[R][64];
  const int r0 = blockIdx.x * R, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, l = tid & 7;
  const int nr = min(R, a.rows - r0);
  if (a.inv_freq) {
    for (int i = tid; i < nr * 64; i += 256) {
      const int r = i >> 6, f = i & 63;
      const double turns =
          static_cast<double>(a.positions[r0 + r]) * static_cast<double>(a.inv_freq[f]) * 0.15915494309189533577;
      double s, c;
      sincospi(2.0 * (turns - rint(turns)), &s, &c);
      cs[r][f] = static_cast<float>(c);
      sn[r][f] = static_cast<float>(s);
    }
    __syncthreads();
  }
  const int Hkv = a.pool.Hkv, nh = a.Hq + 2 * Hkv, quads = (nh + 3) >> 2;
  // the next unit's loads are in flight while one is finished
  auto source = [&](int ri, int quad) {
    return a.qkv + static_cast<size_t>(r0 + ri) * a.ldq + min(4 * quad + (lane >> 3), nh - 1) * 128 + 8 * l;
  };
  auto step = [&](int& ri, int& quad) {  // eight units on
    for (quad += 8; quad >= quads; quad -= quads) ++ri;
  };
  uint4 xl = {}, xh = {};
  int nri = 0, nquad = warp - 8;
  step(nri, nquad);
  if (a.wide && nri < nr) {
    const __nv_bfloat16* src = source(nri, nquad);
    xl = *reinterpret_cast<const uint4*>(src);
    xh = *reinterpret_cast<const uint4*>(src + 64);
  }
  while (nri < nr) {
    const int ri = nri, r = r0 + ri, quad = nquad, h = 4 * quad + (lane >> 3);
    const bool live = h < nh;
    const int hc = live ? h : nh - 1;  // lanes past the last head keep the shuffles whole
    step(nri, nquad);
    float lo[8], hi[8];
    if (a.wide) {
      unpack8(xl, lo);
      unpack8(xh, hi);
      if (nri < nr) {
        const __nv_bfloat16* src = source(nri, nquad);
        xl = *reinterpret_cast<const uint4*>(src);
        xh = *reinterpret_cast<const uint4*>(src + 64);
      }
    } else {
      load8(source(ri, quad), false, lo);
      load8(source(ri, quad) + 64, false, hi);
    }
    const bool is_q = hc < a.Hq, is_v = hc >= a.Hq + Hkv;
    if (a.bias) {
      float bl[8], bh[8];
      load8(a.bias + hc * 128 + 8 * l, a.wide, bl);
      load8(a.bias + hc * 128 + 64 + 8 * l, a.wide, bh);
#pragma unroll
      for (int n = 0; n < 8; ++n) lo[n] += bl[n], hi[n] += bh[n];
    }
    if (a.qnw || a.knw) {
      // pairwise sum of squares: fours of dims, then halves of what is left onto each other
      float f[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float p = __fmul_rn(lo[4 * k], lo[4 * k]), q = __fmul_rn(hi[4 * k], hi[4 * k]);
#pragma unroll
        for (int n = 4 * k + 1; n < 4 * k + 4; ++n) {
          p = __fadd_rn(p, __fmul_rn(lo[n], lo[n]));
          q = __fadd_rn(q, __fmul_rn(hi[n], hi[n]));
        }
        f[k] = __fadd_rn(p, q);
#pragma unroll
        for (int o = 4; o; o >>= 1) f[k] = __fadd_rn(f[k], __shfl_xor_sync(0xffffffffu, f[k], o));
      }
      const float ss = __fadd_rn(f[0], f[1]);
      const __nv_bfloat16* nw = is_q ? a.qnw : a.knw;
      if (!is_v && nw) {
        const float rms = sqrtf(__fadd_rn(ss / 128.0f, a.eps)), inv = 1.0f / rms;
        float wl[8], wh[8];
        load8(nw + 8 * l, a.wide, wl);
        load8(nw + 64 + 8 * l, a.wide, wh);
#pragma unroll
        for (int n = 0; n < 8; ++n) {  // keys become codes: their quotients are exact, q's within an ulp
          lo[n] = __fmul_rn(is_q ? lo[n] * inv : lo[n] / rms, wl[n]);
          hi[n] = __fmul_rn(is_q ? hi[n] * inv : hi[n] / rms, wh[n]);
        }
      }
    }
    if (a.inv_freq && !is_v) {
#pragma unroll
      for (int n4 = 0; n4 < 8; n4 += 4) {
        const float4 c4 = *reinterpret_cast<const float4*>(&cs[ri][8 * l + n4]);
        const float4 s4 = *reinterpret_cast<const float4*>(&sn[ri][8 * l + n4]);
        const float co[4] = {c4.x, c4.y, c4.z, c4.w}, si[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float y = __fsub_rn(__fmul_rn(lo[n4 + n], co[n]), __fmul_rn(hi[n4 + n], si[n]));
          hi[n4 + n] = __fadd_rn(__fmul_rn(hi[n4 + n], co[n]), __fmul_rn(lo[n4 + n], si[n]));
          lo[n4 + n] = y;
        }
      }
    }
    if (is_q && live) {
      __nv_bfloat16* dst = a.q_out + (static_cast<size_t>(r) * a.Hq + hc) * 128 + 8 * l;
      *reinterpret_cast<uint4*>(dst) = pack8(lo);
      *reinterpret_cast<uint4*>(dst + 64) = pack8(hi);
    }
    if (__all_sync(0xffffffffu, is_q)) continue;
    // every lane of the warp reduces (another eight may hold a key)
    uint32_t ml = 0, mh = 0;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      ml = max(ml, __float_as_uint(fabsf(lo[n])));
      mh = max(mh, __float_as_uint(fabsf(hi[n])));
    }
    ml = group_max(ml);
    mh = group_max(mh);
    const int slot = a.slots[r];
    if (is_q || !live || slot < 0) continue;
    const int b = a.seq ? a.seq[r] : r / a.rows_per_seq;
    uint8_t* dst = a.pool.block_of(b, slot, a.err, l == 0);
    if (!dst) continue;
    dst += static_cast<size_t>(hc - a.Hq - (is_v ? Hkv : 0)) * a.pool.hstride();
    const int in = slot & 15, j = l >> 2;
    const __half sl = group_scale(ml), sh = group_scale(mh);
    const uint32_t wl = eight_codes(lo, __half2float(sl)), wh = eight_codes(hi, __half2float(sh));
    if (is_v) {
      *reinterpret_cast<uint16_t*>(dst + v_code_offset(in, 2 * l)) = static_cast<uint16_t>(wl);
      *reinterpret_cast<uint16_t*>(dst + v_code_offset(in, 2 * l + 1)) = static_cast<uint16_t>(wl >> 16);
      *reinterpret_cast<uint16_t*>(dst + v_code_offset(in, 2 * l + 16)) = static_cast<uint16_t>(wh);
      *reinterpret_cast<uint16_t*>(dst + v_code_offset(in, 2 * l + 17)) = static_cast<uint16_t>(wh >> 16);
    } else {
      *reinterpret_cast<uint32_t*>(dst + k_code_offset(in, 2 * l)) = wl;
      *reinterpret_cast<uint32_t*>(dst + k_code_offset(in, 2 * l + 16)) = wh;
    }
    if ((l & 3) == 0) {
      *reinterpret_cast<__half*>(dst + (is_v ? v_scale_offset(in, j) : k_scale_offset(in, j))) = sl;
      *reinterpret_cast<__half*>(dst + (is_v ? v_scale_offset(in, j + 2) : k_scale_offset(in, j + 2))) = sh;
    }
  }
}

// Read-back of listed slots as bf16 rows: eight lanes per (row, kv head), as in the append.
__global__ void __launch_bounds__(256) gather_kernel(const int* __restrict__ slots, const int* __restrict__ seq,
                                                     int rows_per_seq, int rows, Pool pool,
                                                     __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out,
                                                     long long row_stride, long long head_stride, int* err) {
  pdl_launch_dependents();
  pdl_wait();
  const unsigned r = blockIdx.x * 32 + (threadIdx.x >> 3);
  const int l = threadIdx.x & 7, h = blockIdx.y;
  if (r >= static_cast<unsigned>(rows)) return;
  const int slot = slots[r];
  const int b = seq ? seq[r] : static_cast<int>(r) / rows_per_seq;
  const uint8_t* blk = slot >= 0 ? pool.block_of(b, slot, err, h == 0 && l == 0) : nullptr;
  uint4 o[4] = {};
  if (blk) {
    blk += h * pool.hstride();
    const int in = slot & 15, j = l >> 2;
    auto u16 = [&](int at) { return static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(blk + at)); };
    const uint32_t w[4] = {*reinterpret_cast<const uint32_t*>(blk + k_code_offset(in, 2 * l)),
                           *reinterpret_cast<const uint32_t*>(blk + k_code_offset(in, 2 * l + 16)),
                           u16(v_code_offset(in, 2 * l)) | u16(v_code_offset(in, 2 * l + 1)) << 16,
                           u16(v_code_offset(in, 2 * l + 16)) | u16(v_code_offset(in, 2 * l + 17)) << 16};
    const float s[4] = {__half2float(__ushort_as_half(u16(k_scale_offset(in, j)))),
                        __half2float(__ushort_as_half(u16(k_scale_offset(in, j + 2)))),
                        __half2float(__ushort_as_half(u16(v_scale_offset(in, j)))),
                        __half2float(__ushort_as_half(u16(v_scale_offset(in, j + 2))))};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = static_cast<float>(static_cast<int>((w[i] >> (4 * k)) & 15u) - 8) * s[i];
      o[i] = pack8(x);
    }
  }
  const long long at = r * row_stride + h * head_stride + 8 * l;
  *reinterpret_cast<uint4*>(k_out + at) = o[0];
  *reinterpret_cast<uint4*>(k_out + at + 64) = o[1];
  *reinterpret_cast<uint4*>(v_out + at) = o[2];
  *reinterpret_cast<uint4*>(v_out + at + 64) = o[3];
}

// ---- attention of one token per sequence ------------------------------------------------
// softmax(scale q . k) v for the <= 8 query heads of a kv head, slots on the M side of
// mma.sync m16n8k16 (f16 operands, fp32 sums) and heads on N.
//
// What bounds it: HBM, 144 bytes per slot and kv head -- 46 codes per clock and SM at the
// copy bandwidth, so unpacking has to cost about one instruction per code:
//  * integers become floats by the published method of or-ing them into the mantissa of a fixed
//    exponent, which 4-bit weight products use too: (word & 0x000f000f) | 0x64006400 is the f16
//    pair 1024 + n, (word & 0x00f000f0) | 0x64006400 the pair 1024 + 16 n; one packed add or
//    multiply-add makes either the exact code n - 8: 9 instructions per 8 codes.  (Feeding the MMA
//    the biased pairs, or the bare bits as f16 subnormals, and taking the bias off the sums saves
//    4 of the 9 but not the precision: the MMA aligns products by their operands' exponent fields,
//    10 bits above the code's own, and its sums came out 2^-16 off.)
//  * scales never touch the codes: K's multiply the four group sums in fp32, V's multiply the
//    softmax weights (P' = P * scale, f16, rounded at 2^-11: half a bf16 output step is 2^-9).
// P is 2^(x - ref), ref = max(x) - kTop at least and moved only when the maximum has grown by
// kSlack bits: the largest P is 2^10 to 2^14, so P's smallest step is 2^-34 of the largest weight
// or finer.  V's scales are brought near 1 by a power of two for each group of 32 dims (taken off
// O at the end), from the largest scale of the group's live slots: a product's smallest step is
// 2^-29 of that scale times the largest weight or finer, whatever the other groups hold (2^-48
// times the weight where all of the group's scales are subnormal).  One exponent for all groups
// would cost quiet ones beside a loud one their bits.
// q is brought to [2^14, 2^15) by a power of two for the same reason (exact: q is bf16).
// A masked slot's logit is -inf and its V scale zero, so nothing it holds (NaN scales of
// never-written memory included) reaches a sum; codes are finite whatever their bits.
//
// Work split: the 16-slot blocks of all sequences and heads in one line, cut into equal
// ranges, one per CTA (two CTAs of 8 warps per SM), whatever the lengths.  A range crosses
// heads; within a head's part ("segment") the warps take turns at 32-slot stages, each warp
// with its own two-stage ring of bulk copies that runs on across segments, so no barrier
// stands in the stream.  At the end of a segment the warps' (ref, sum, O) meet in shared
// memory; a whole head is written out, a part of one goes to the workspace (at most two per
// CTA) for the combine kernel.  Logits for the eviction score go to the workspace too: the
// probabilities need the final (ref, sum).
//
// Measured: 8 kv heads of one sequence of 131071 slots 46.8 us (3.2 TB/s, 23.1 at the copy
// bandwidth), 64 sequences x 8 heads of 4104 slots with masks and score 103 us (47); 7 % more where
// V's scales lie outside [2^-5, 2) (20 % in the one-launch form below).  The copies alone, with the
// arithmetic skipped, take 36 and 64 us; the rest is issue: 365 instructions per block and warp
// against 250 that the arithmetic needs, 61 % of the issue slots used (16 warps at 128 registers).
// Slower: four-block stages and 8 warps (289 instructions, but 50 % of the
// slots: 46 and 112 us), 12 or 16 warps in one CTA (49 / 109, 49 / 110), one CTA of 8 warps with
// two-block stages (53 / 125).
constexpr int kWarps = 8;
constexpr int kStages = 2;       // per warp
constexpr int kStageBlocks = 2;  // 16-slot blocks per stage
constexpr int kCtas = 2;         // per SM
constexpr float kTop = 14.f;     // the largest weight is 2^kTop at most, and P' below twice that
constexpr float kSlack = 4.f;    // how far (in bits) the running maximum may grow before a rescale
constexpr int kMaxSeqs = 256;    // sequences per launch (their lengths live in shared memory)
constexpr int kMaxCtas = 320;
constexpr int kMinBlocks = 2 * kWarps;  // blocks per CTA at least
constexpr int kHeadPitch = 132;  // floats between heads of a partial O (conflict-free float4 stores)
constexpr int kPart = 8 * 128 + 16;  // floats of one partial: O[8][128], ref[8], sum[8]

// Workspace: int header[2 + kMaxSeqs + 1] {blocks per CTA, -, first block of each sequence},
// partials [kMaxCtas][2][kPart], and with a score the whole heads' (ref, sum) [B][Hkv][8][2]
// and the logits [B][Hkv][S16][gs] in units of ln 2.
constexpr size_t kHeaderBytes = ((2 + kMaxSeqs + 1) * 4 + 15) / 16 * 16;
constexpr size_t kPartBytes = static_cast<size_t>(kMaxCtas) * 2 * kPart * 4;

struct AttnArgs {
  const __nv_bfloat16* q;
  Pool pool;
  const int* lens;
  const int* slot_pos;
  __nv_bfloat16* out;
  float* step_score;
  int* header;
  float* part;
  float* stats;   // null without a score
  float* logits;  // null without a score
  int* err;
  float scale;
  int Hq, S, limit;
  int s16, gs;  // logit rows per head, floats per row
};

// The powers of two that a warp takes V's scales by, group by group: scale * 2^-k.
struct Moves {
  uint4 shrink;  // 2^-k as f16 pairs
  int k[4];
};

struct Smem {
  uint8_t ring[kWarps][kStages][kStageBlocks * kBlock];
  float part[kWarps][8][kHeadPitch];
  float ref[kWarps][8], sum[kWarps][8];
  uint4 q[2][4][32];  // a head's B operands: [parity of the segment][group][lane]
  float xs[2][8];     // and its logits per unit of the MMAs' sums
  Moves moves[kWarps];
  uint64_t full[kWarps][kStages];
  int first[kMaxSeqs + 1];  // first block of each sequence's first head
  int len[kMaxSeqs];
  int wsum[kWarps], wmax[kWarps];
};
static_assert(sizeof(Smem) <= 115712 - 16, "two CTAs per SM");

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with a zero accumulator
__device__ __forceinline__ void mma_f16_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The codes n - 8 of nibbles 0 and 4 / 1 and 5 of a word, as f16 pairs for the MMA.
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(r) : "r"(w));
  const uint32_t c = 0xe408e408u;  // -1032
  asm("add.rn.f16x2 %0, %0, %1;" : "+r"(r) : "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t code_pair_hi(uint32_t w) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(r) : "r"(w));
  const uint32_t m = 0x2c002c00u, c = 0xd480d480u;  // 1 / 16, -72
  asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(r) : "r"(m), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_half2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

__device__ __forceinline__ float pow2(int k) { return __int_as_float((127 + k) << 23); }

// What a warp has of its slots' softmax: per query head (columns 2 t, 2 t + 1 of the MMAs) the
// reference exponent and this thread's share of the sum, and O in the MMAs' layout: thread
// (g, t) holds dims 32 i + 4 g + {0, 1, 2, 3} of the two heads in o[2 i][0, 1], o[2 i][2, 3],
// o[2 i + 1][0, 1], o[2 i + 1][2, 3].
struct Sums {
  float o[8][4], l[2], ref[2];
  bool moved;  // some of this warp's k are not 0 (else none is written)
  Moves* mv;
  __device__ __forceinline__ void clear(Moves* to) {
    mv = to;
    moved = false;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
    l[0] = l[1] = 0.f;
    ref[0] = ref[1] = -INFINITY;
  }
  // a slot pair's V scales of all groups, or of groups 2 half and 2 half + 1, times 2^-k
  __device__ __forceinline__ uint4 scaled(uint4 v) const {
    const uint4 by = mv->shrink;
    v.x = half2_bits(__hmul2(bits_half2(v.x), bits_half2(by.x)));
    v.y = half2_bits(__hmul2(bits_half2(v.y), bits_half2(by.y)));
    v.z = half2_bits(__hmul2(bits_half2(v.z), bits_half2(by.z)));
    v.w = half2_bits(__hmul2(bits_half2(v.w), bits_half2(by.w)));
    return v;
  }
  __device__ __forceinline__ uint2 scaled(uint2 v, int half) const {
    const uint2 by = reinterpret_cast<const uint2*>(&mv->shrink)[half];
    v.x = half2_bits(__hmul2(bits_half2(v.x), bits_half2(by.x)));
    v.y = half2_bits(__hmul2(bits_half2(v.y), bits_half2(by.y)));
    return v;
  }
  // Rescale where a weight would pass 2^kTop, then with kSlack bits to spare, or a scale is 2 or
  // more: most stages only vote.  ``bits``: the warp's live scales as they would enter the
  // products, or-ed (only those from 2 on have bit 14); most(m) leaves this lane's largest scales
  // as stored of each group.  True when k is another than before.
  template <typename Most>
  __device__ __forceinline__ bool vote(float (&top)[2], uint32_t bits, int lane, Most most) {
    if (!__any_sync(0xffffffffu, (bits & 0x40004000u) || top[0] - ref[0] > kTop || top[1] - ref[1] > kTop)) return false;
    const bool fresh = !__any_sync(0xffffffffu, ref[0] > -INFINITY || ref[1] > -INFINITY);  // O is empty
    // The largest scale of each group, as bits (they order like integers; a NaN makes its own
    // group NaN whatever k).  Those in [2^-5, 2) stay as they are, so that ordinary values cost no
    // more than this vote; others go to [1, 2).  k only grows.
    uint32_t m[4], flags = bits & 0x40004000u ? 16u : 0u;
    most(m);
#pragma unroll
    for (int i = 0; i < 4; ++i) flags |= m[i] >= 10u << 10 ? 1u << i : 0u;
    flags = __reduce_or_sync(0xffffffffu, flags);
    const bool move = flags >= 16u || (fresh && flags != 15u);
    if (move) {
      int now[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int f = min(30, static_cast<int>(__reduce_max_sync(0xffffffffu, m[i]) >> 10));
        const int was = moved ? mv->k[i] : 0;
        now[i] = f >= 10 && f <= 15 ? 0 : f - 15;
        if (!fresh) now[i] = max(now[i], was);
        const float g = pow2(was - now[i]);
#pragma unroll
        for (int c = 0; c < 4; ++c) o[2 * i][c] *= g, o[2 * i + 1][c] *= g;
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane == i) {
          mv->k[i] = now[i];  // 2^-15 is subnormal
          reinterpret_cast<uint32_t*>(&mv->shrink)[i] = (now[i] < 15 ? static_cast<uint32_t>(15 - now[i]) << 10 : 0x200u) * 0x10001u;
        }
      __syncwarp();
      moved = true;
    }
    float f[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 4));
      top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 8));
      top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 16));
      // differences are exact where they are small, sums round: from 2^26 on, top - 10 may lie
      // 16 below top (there the next smaller weight is 2^-8 of this one at most)
      float r = top[c] - ref[c] > kTop ? top[c] - (kTop - kSlack) : ref[c];
      if (top[c] - r > kTop) r = top[c];
      f[c] = r == ref[c] ? 1.0f : ex2(ref[c] - r);  // also where both are -inf
      ref[c] = r;
      l[c] *= f[c];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i][0] *= f[0], o[i][1] *= f[1], o[i][2] *= f[0], o[i][3] *= f[1];
    return move;
  }
  // O += P V of a block: its logits x, V codes (v0, v1) and V scales (s0, s1) of the slot pairs
  __device__ __forceinline__ void weigh(const float (&x)[4], const uint4 v0, const uint4 v1, const uint4 s0, const uint4 s1) {
    const float r0 = ref[0] == -INFINITY ? 0.f : ref[0], r1 = ref[1] == -INFINITY ? 0.f : ref[1];
    const float p0 = ex2(x[0] - r0), p1 = ex2(x[1] - r1), p2 = ex2(x[2] - r0), p3 = ex2(x[3] - r1);
    l[0] += p0 + p2;
    l[1] += p1 + p3;
    const __half2 b0 = bits_half2(transpose8x8(half2_bits(__floats2half2_rn(p0, p1))));
    const __half2 b1 = bits_half2(transpose8x8(half2_bits(__floats2half2_rn(p2, p3))));
    const uint32_t sa[4] = {s0.x, s0.y, s0.z, s0.w}, sb[4] = {s1.x, s1.y, s1.z, s1.w};
    const uint32_t w0[4] = {v0.x, v0.y, v0.z, v0.w}, w1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t c0 = half2_bits(__hmul2(b0, bits_half2(sa[i]))), c1 = half2_bits(__hmul2(b1, bits_half2(sb[i])));
      const uint32_t u0 = w0[i] >> 8, u1 = w1[i] >> 8;
      mma_f16(o[2 * i], code_pair(w0[i]), code_pair_hi(w0[i]), code_pair(w1[i]), code_pair_hi(w1[i]), c0, c1);
      mma_f16(o[2 * i + 1], code_pair(u0), code_pair_hi(u0), code_pair(u1), code_pair_hi(u1), c0, c1);
    }
  }
  // the warp's sums to shared memory: ref and sum [8], O [8][kHeadPitch] of the live heads
  __device__ __forceinline__ void leave(float* to_ref, float* to_sum, float (*to_o)[kHeadPitch], int group, bool any, int g, int t) {
    if (moved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = pow2(mv->k[i >> 1]);
#pragma unroll
        for (int c = 0; c < 4; ++c) o[i][c] *= u;
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      l[c] += __shfl_xor_sync(0xffffffffu, l[c], 4);
      l[c] += __shfl_xor_sync(0xffffffffu, l[c], 8);
      l[c] += __shfl_xor_sync(0xffffffffu, l[c], 16);
      if (g == 0) to_ref[2 * t + c] = ref[c], to_sum[2 * t + c] = l[c];
      if (any && 2 * t + c < group) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(&to_o[2 * t + c][32 * i + 4 * g]) =
              make_float4(o[2 * i][c], o[2 * i][c + 2], o[2 * i + 1][c], o[2 * i + 1][c + 2]);
      }
    }
  }
};
// Logits (in units of ln 2) of a block's slots sg (x[0, 1]) and sg + 2 (x[2, 3]) for heads 2 t,
// 2 t + 1: K codes and scales of the two slots; q(j) is group j's B operand.
template <typename Q>
__device__ __forceinline__ void block_logits(const uint4 k0, const uint4 k1, const uint2 s0, const uint2 s1, Q q,
                                             const float (&xs)[2], float (&x)[4]) {
  const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
  const float2 f0[2] = {__half22float2(bits_half2(s0.x)), __half22float2(bits_half2(s0.y))};
  const float2 f1[2] = {__half22float2(bits_half2(s1.x)), __half22float2(bits_half2(s1.y))};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float c[4];
    const uint4 qf = q(j);
    const uint32_t u0 = w0[j] >> 8, u1 = w1[j] >> 8;
    mma_f16_new(c, code_pair(w0[j]), code_pair(w1[j]), code_pair_hi(w0[j]), code_pair_hi(w1[j]), qf.x, qf.y);
    mma_f16(c, code_pair(u0), code_pair(u1), code_pair_hi(u0), code_pair_hi(u1), qf.z, qf.w);
    const float a0 = j & 1 ? f0[j >> 1].y : f0[j >> 1].x, a1 = j & 1 ? f1[j >> 1].y : f1[j >> 1].x;
    x[0] = j ? x[0] + a0 * c[0] : a0 * c[0];
    x[1] = j ? x[1] + a0 * c[1] : a0 * c[1];
    x[2] = j ? x[2] + a1 * c[2] : a1 * c[2];
    x[3] = j ? x[3] + a1 * c[3] : a1 * c[3];
  }
  x[0] *= xs[0];
  x[1] *= xs[1];
  x[2] *= xs[0];
  x[3] *= xs[1];
}
__device__ __forceinline__ uint32_t or4(const uint4 v) { return v.x | v.y | v.z | v.w; }
__device__ __forceinline__ uint32_t max_half(uint32_t pair) { return max(pair & 0x7fffu, pair >> 16 & 0x7fffu); }
// -inf for the masked ones of slots sg and sg + 2 (bits 0 and 2 of m)
__device__ __forceinline__ void mask_logits(float (&x)[4], uint32_t m) {
  if (!(m & 1u)) x[0] = x[1] = -INFINITY;
  if (!(m & 4u)) x[2] = x[3] = -INFINITY;
}
// the V scales of a slot pair, zero where masked (the memory may hold anything)
__device__ __forceinline__ uint32_t pair_mask(uint32_t two) {
  return (two & 1u ? 0x0000ffffu : 0u) | (two & 2u ? 0xffff0000u : 0u);
}
__device__ __forceinline__ uint4 mask_scales(uint4 v, uint32_t two) {
  const uint32_t keep = pair_mask(two);
  v.x &= keep, v.y &= keep, v.z &= keep, v.w &= keep;
  return v;
}
// q of head g (zeros where not live) as the MMA's B operands, group j in qf[j], brought to
// [2^14, 2^15) by 2^up; returns the head's logits in units of ln 2 per unit of the MMAs' sums:
// scale log2(e) / 2^up, in two factors (2^-up alone can overflow).
__device__ __forceinline__ float load_query(const __nv_bfloat16* head, bool live, float scale, int t, uint4 (&qf)[4]) {
  const uint4* src = reinterpret_cast<const uint4*>(head);
  uint4 w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = live ? src[4 * j + t] : make_uint4(0, 0, 0, 0);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t ws[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) top = max(top, max((ws[k] >> 16) & 0x7fffu, ws[k] & 0x7fffu));
  }
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int up = min(14 + 127 - static_cast<int>(top >> 7), 126);
  const float f = __int_as_float((up + 127) << 23);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float d[8] = {bf16lo(w[j].x) * f, bf16hi(w[j].x) * f, bf16lo(w[j].y) * f, bf16hi(w[j].y) * f,
                        bf16lo(w[j].z) * f, bf16hi(w[j].z) * f, bf16lo(w[j].w) * f, bf16hi(w[j].w) * f};
    qf[j] = make_uint4(half2_bits(__floats2half2_rn(d[0], d[4])), half2_bits(__floats2half2_rn(d[1], d[5])),
                       half2_bits(__floats2half2_rn(d[2], d[6])), half2_bits(__floats2half2_rn(d[3], d[7])));
  }
  return scale * 1.4426950408889634f * __int_as_float((127 - (up >> 1)) << 23) *
         __int_as_float((127 - (up - (up >> 1))) << 23);
}

// A range's part of one (sequence, kv head): blocks [sb0, sb0 + n) of the head's nsb.
struct Segment {
  int b, h, sb0, n, nsb;
  __device__ __forceinline__ void at(const Smem& sm, int Hkv, int pos, int end) {  // b: any sequence at or before pos
    while (sm.first[b + 1] <= pos) ++b;
    nsb = (sm.len[b] + 15) >> 4;
    const int o = pos - sm.first[b];
    h = o / nsb;
    sb0 = o - h * nsb;
    n = min(nsb - sb0, end - pos);
  }
  // blocks per stage: short segments are spread over all warps
  __device__ __forceinline__ int per() const {
    return n <= kWarps ? 1 : kStageBlocks;
  }
};

// The lengths' prefix sums into shared memory; returns the number of blocks of all heads, and
// of the longest one.
__device__ __forceinline__ int plan(const AttnArgs& a, Smem& sm, bool report, int& longest) {
  const int B = a.pool.B, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kEach = (kMaxSeqs + kWarps * 32 - 1) / (kWarps * 32);
  int v[kEach], t = 0, most = 0;
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const int b = tid * kEach + u;
    int n = b < B ? a.lens[b] : 0;
    if (n < 0 || n > a.limit) {
      if (report) set_err(a.err, kErrIndex);
      n = n < 0 ? 0 : a.limit;
    }
    if (b < B) sm.len[b] = n;
    v[u] = t;
    t += ((n + 15) >> 4) * a.pool.Hkv;
    most = max(most, (n + 15) >> 4);
  }
  int inc = t;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 31) sm.wsum[warp] = inc, sm.wmax[warp] = most;
  __syncthreads();
  int before = 0, total = 0;
  longest = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    longest = max(longest, sm.wmax[w]);
    if (w < warp) before += sm.wsum[w];
    total += sm.wsum[w];
  }
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const int b = tid * kEach + u;
    if (b < B) sm.first[b] = before + inc - t + v[u];
  }
  if (tid == 0) sm.first[B] = total;
  __syncthreads();
  return total;
}

template <bool kScore>
__global__ void __launch_bounds__(kWarps * 32, kCtas) attend_kernel(const AttnArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int Hkv = a.pool.Hkv, group = a.Hq / Hkv;
  if (lane == 0)
    for (int s = 0; s < kStages; ++s) mbar_init(&sm.full[warp][s], 1);
  fence_barrier_init();
  pdl_launch_dependents();
  pdl_wait();
  int longest;
  const int total = plan(a, sm, blockIdx.x == 0, longest);
  // at least kMinBlocks of a head, or short heads one after the other would wait in few CTAs
  const int R = max((total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x), min(kMinBlocks, longest));
  if (blockIdx.x == 0) {
    if (tid == 0) a.header[0] = R;
    for (int b = tid; b <= a.pool.B; b += kWarps * 32) a.header[2 + b] = sm.first[b];
  }
  const int start = static_cast<int>(min(static_cast<long long>(blockIdx.x) * R, static_cast<long long>(total)));
  const int end = min(total - start, R) + start;
  if (start >= end) return;

  // -- the stage to be issued next is found one stage ahead, so that its page and mask loads
  //    are not waited for; lane i < cnt follows the stage's block i (page index pi, block
  //    ``inner`` of the page), which moves by whole turns of the warps within a segment
  const int ppb = a.pool.page >> 4;  // blocks per page
  constexpr int kTurn = kWarps * kStageBlocks;
  const int turn_pages = kTurn / ppb, turn_inner = kTurn - turn_pages * ppb;
  Segment is;
  {
    int lo = 0, hi = a.pool.B - 1;  // the last sequence that starts at or before ``start``
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sm.first[mid] <= start) lo = mid;
      else hi = mid - 1;
    }
    is.b = lo;
  }
  is.at(sm, Hkv, start, end);
  Segment cs = is;
  int ipos = start, left;  // left: blocks of the segment from this warp's stage on
  bool have = true, live;
  int slot, pi, inner, cnt, page;
  uint32_t masks[kStages];  // live slots of the stages in the ring
  auto enter = [&]() {  // this warp's first stage of segment ``is``
    const int k = warp * is.per();
    left = is.n - k;
    slot = (is.sb0 + k) * 16 + lane;
    const int blk = is.sb0 + k + (lane < kStageBlocks ? lane : 0);
    pi = blk / ppb;
    inner = blk - pi * ppb;
  };
  auto look = [&]() {  // at the stage ``left`` points to, or the next segment's first
    while (left <= 0) {
      ipos += is.n;
      if (ipos >= end) {
        have = false;
        return;
      }
      is.at(sm, Hkv, ipos, end);
      enter();
    }
    cnt = min(is.per(), left);
    live = lane < cnt * 16 && slot < sm.len[is.b];
    if (a.slot_pos && live) live = a.slot_pos[static_cast<size_t>(is.b) * a.S + slot] >= 0;
    page = lane < cnt ? a.pool.table[static_cast<size_t>(is.b) * a.pool.max_pages + pi] : -1;
  };
  auto issue = [&](int st) {  // the stage last looked at, and on to the next
    if (!have) return;
    const bool ok = static_cast<unsigned>(page) < static_cast<unsigned>(a.pool.n_pages);
    const uint32_t okm = __ballot_sync(0xffffffffu, ok);
    uint32_t mask = __ballot_sync(0xffffffffu, live);
    if (okm != (1u << cnt) - 1u) {  // a page out of range: its slots are masked
      if (lane < cnt && !ok) set_err(a.err, kErrIndex);
      mask &= (okm & 1u ? 0x0000ffffu : 0u) | (okm & 2u ? 0xffff0000u : 0u);
    }
#pragma unroll
    for (int s = 0; s < kStages; ++s) masks[s] = s == st ? mask : masks[s];
    if (lane == 0) mbar_expect_tx(&sm.full[warp][st], __popc(okm) * kBlock);
    __syncwarp();
    if (ok)
      bulk_load(sm.ring[warp][st] + lane * kBlock,
                a.pool.base + ((static_cast<size_t>(page) * Hkv + is.h) * ppb + inner) * kBlock, kBlock,
                &sm.full[warp][st]);
    left -= kWarps * is.per();  // a segment of smaller stages has one turn only
    slot += kTurn * 16;
    pi += turn_pages;
    inner += turn_inner;
    if (inner >= ppb) inner -= ppb, ++pi;
    look();
  };
  enter();
  look();
#pragma unroll
  for (int s = 0; s < kStages; ++s) issue(s);

  auto prepare_q = [&](const Segment& s, int buf) {  // q of a segment's head: one warp's work
    uint4 qf[4];
    const float unit = load_query(a.q + (static_cast<size_t>(s.b) * a.Hq + s.h * group + g) * 128, g < group, a.scale, t, qf);
#pragma unroll
    for (int j = 0; j < 4; ++j) sm.q[buf][j][lane] = qf[j];
    if (t == 0) sm.xs[buf][g] = unit;
  };
  if (warp == kWarps - 1) prepare_q(cs, 0);
  __syncthreads();

  int st = 0, phase = 0, buf = 0;  // the stage consumed next; the segment's q
  bool dead = false;               // a copy never arrived: stop streaming, keep the barriers
  const int sg = 4 * (g >> 1) + (g & 1);  // slot (of 16) of MMA row g; row g + 8 is slot sg + 2
  for (int pos = start; pos < end;) {
    Segment next = cs;
    if (pos + cs.n < end) {
      next.at(sm, Hkv, pos + cs.n, end);
      if (warp == kWarps - 1) prepare_q(next, buf ^ 1);
    }
    const float xs[2] = {sm.xs[buf][2 * t], sm.xs[buf][2 * t + 1]};
    Sums sums;
    sums.clear(&sm.moves[warp]);
    auto q_of = [&](int j) { return sm.q[buf][j][lane]; };

    const int per = cs.per();
    float* lg = kScore && 2 * t < a.gs
                    ? a.logits + (static_cast<size_t>(cs.b * Hkv + cs.h) * a.s16 + cs.sb0 * 16 + sg) * a.gs + 2 * t
                    : nullptr;
    for (int k = warp * per; k < cs.n; k += kWarps * per) {
      const int nb = min(per, cs.n - k);
      if (!dead && !__all_sync(0xffffffffu, mbar_wait_bounded(&sm.full[warp][st], phase))) {
        dead = true;  // let the other stages' copies land before the CTA can exit
        if (lane == 0) set_err(a.err, kErrWaitTimeout);
        for (int s = 1; s < kStages; ++s)
          mbar_wait_bounded(&sm.full[warp][(st + s) % kStages], phase ^ (st + s >= kStages), 1u << 16);
        __syncwarp();
      }
      uint32_t mask = masks[0];
#pragma unroll
      for (int s = 1; s < kStages; ++s) mask = s == st ? masks[s] : mask;
      if (dead) mask = 0;
      uint8_t* base = sm.ring[warp][st];
      auto process = [&](auto full_stage) {
        constexpr bool kFull = decltype(full_stage)::value;  // no mask, no missing block
        auto v_scales = [&](int bl, int h) {  // of this thread's slot pair 4 t + 2 h
          const uint4 v = *reinterpret_cast<const uint4*>(base + bl * kBlock + kVScale + 32 * t + 16 * h);
          return kFull ? v : mask_scales(v, mask >> (16 * bl + 4 * t + 2 * h));
        };
        float x[kStageBlocks][4], top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int bl = 0; bl < kStageBlocks; ++bl) {
          if (!kFull && bl >= nb) break;
          const uint8_t* blk = base + bl * kBlock;
          block_logits(*reinterpret_cast<const uint4*>(blk + 64 * sg + 16 * t),
                       *reinterpret_cast<const uint4*>(blk + 64 * (sg + 2) + 16 * t),
                       *reinterpret_cast<const uint2*>(blk + kKScale + 8 * sg),
                       *reinterpret_cast<const uint2*>(blk + kKScale + 8 * (sg + 2)), q_of, xs, x[bl]);
          if (!kFull) mask_logits(x[bl], mask >> (16 * bl + sg));
          if (kScore && lg) {
            float* to = lg + (k + bl) * 16 * a.gs;
            *reinterpret_cast<float2*>(to) = make_float2(x[bl][0], x[bl][1]);
            *reinterpret_cast<float2*>(to + 2 * a.gs) = make_float2(x[bl][2], x[bl][3]);
          }
          top[0] = fmaxf(top[0], fmaxf(x[bl][0], x[bl][2]));
          top[1] = fmaxf(top[1], fmaxf(x[bl][1], x[bl][3]));
        }
        // lane 16 bl + 4 t + 2 h + p has the stage's V scales of slots 4 t + 2 h and the next of
        // block bl, groups 2 p and 2 p + 1
        static_assert(kStageBlocks == 2, "a lane's two words");
        uint2* two = reinterpret_cast<uint2*>(base + (lane >> 4) * kBlock + kVScale) + (lane & 15);
        const uint32_t keep = kFull ? 0xffffffffu : pair_mask(mask >> (lane & 30));
        uint2 w = *two;
        if (sums.moved) w = sums.scaled(w, lane & 1);
        sums.vote(top, (w.x | w.y) & keep, lane, [&](uint32_t (&m)[4]) {
          const uint2 v = *two;
          const uint32_t a = max_half(v.x & keep), b = max_half(v.y & keep);
          m[0] = lane & 1 ? 0u : a, m[1] = lane & 1 ? 0u : b, m[2] = lane & 1 ? a : 0u, m[3] = lane & 1 ? b : 0u;
        });
        if (sums.moved) {  // the products below find them scaled
          *two = sums.scaled(*two, lane & 1);
          fence_proxy_async_smem();  // the next copy into the stage comes after these writes
          __syncwarp();
        }
#pragma unroll
        for (int bl = 0; bl < kStageBlocks; ++bl) {
          if (!kFull && bl >= nb) break;
          const uint8_t* blk = base + bl * kBlock;
          sums.weigh(x[bl], *reinterpret_cast<const uint4*>(blk + 1024 + 64 * g + 16 * t),
                     *reinterpret_cast<const uint4*>(blk + 1536 + 64 * g + 16 * t), v_scales(bl, 0), v_scales(bl, 1));
        }
      };
      if (mask == 0xffffffffu) process(std::true_type{});  // every slot of a whole stage is live
      else process(std::false_type{});
      __syncwarp();
      if (!dead) issue(st);
      if (++st == kStages) st = 0, phase ^= 1;
    }

    // -- the warps' parts of this segment meet
    sums.leave(sm.ref[warp], sm.sum[warp], sm.part[warp], group, warp * per < cs.n, g, t);
    __syncthreads();
    const bool whole = cs.n == cs.nsb;
    if (warp < group) {  // one query head per warp, four dims per lane
      float M = -INFINITY, L = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm.ref[w][warp]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float rw = sm.ref[w][warp];
        const float lw = sm.sum[w][warp];
        if (rw > -INFINITY || lw != 0.f) {  // also a NaN sum
          const float fw = rw == M ? 1.0f : ex2(rw - M);
          const float4 v = *reinterpret_cast<const float4*>(&sm.part[w][warp][4 * lane]);
          L += lw * fw;
          acc.x += v.x * fw, acc.y += v.y * fw, acc.z += v.z * fw, acc.w += v.w * fw;
        }
      }
      if (whole) {
        const bool none = L == 0.f;
        const float r = none ? 0.f : 1.0f / L;
        __nv_bfloat16* dst = a.out + (static_cast<size_t>(cs.b) * a.Hq + cs.h * group + warp) * 128 + 4 * lane;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc.x * r, acc.y * r), pack_bf16(acc.z * r, acc.w * r));
        if (lane == 0) {
          if (none) set_err(a.err, kErrNoValidSlot);
          if (a.stats) {
            float* s = a.stats + (static_cast<size_t>(cs.b * Hkv + cs.h) * 8 + warp) * 2;
            s[0] = M;
            s[1] = L;
          }
        }
      } else {
        float* p = a.part + (static_cast<size_t>(blockIdx.x) * 2 + (pos == start ? 0 : 1)) * kPart;
        *reinterpret_cast<float4*>(p + warp * 128 + 4 * lane) = acc;
        if (lane == 0) p[1024 + warp] = M, p[1032 + warp] = L;
      }
    }
    pos += cs.n;
    cs = next;
    buf ^= 1;
    // the parts have been read, so the next segment may write its own; its q is in place
    if (pos < end) __syncthreads();
  }
}

// Finishes what the streaming kernel left: CTAs x < ceil(Hq / 2) join the parts of two query
// heads of a sequence (or write zeros for an empty one), four warps a head with a quarter of
// the parts each; the others form the eviction score of 256 slots of a sequence from the
// logits and the final (ref, sum) of its heads.  One launch for both: they are short and
// latency-bound, so loads are issued as early and as many as possible.
__global__ void __launch_bounds__(256) combine_kernel(const AttnArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ float2 fin[];  // (ref, 1 / sum) of every query head of the sequence
  __shared__ float4 quarter[8][32];
  __shared__ float2 qsum[8];
  const int Hkv = a.pool.Hkv, group = a.Hq / Hkv, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int R = a.header[0], first = a.header[2 + b], nsb = (a.header[2 + b + 1] - first) / Hkv;
  // the part of head (b, h), first block s0, that CTA c left: in the CTA's first place where
  // the CTA's range starts inside the head
  auto part_of = [&](int c, int s0) {
    return a.part + (static_cast<size_t>(c) * 2 + (c * static_cast<long long>(R) >= s0 ? 0 : 1)) * kPart;
  };
  auto join = [](float& M, float& L, float m, float l) {  // (M, L) += (m, l)
    const float top = fmaxf(M, m);
    L = L * (M == top ? 1.0f : ex2(M - top)) + l * (m == top ? 1.0f : ex2(m - top));
    M = top;
  };
  const int pairs = (a.Hq + 1) >> 1;
  if (static_cast<int>(blockIdx.x) < pairs) {
    const int q = min(2 * static_cast<int>(blockIdx.x) + (warp >> 2), a.Hq - 1), mine = warp & 3;
    const int h = q / group, w = q - h * group;
    const int s0 = first + h * nsb, c0 = nsb ? s0 / R : 0, c1 = nsb ? (s0 + nsb - 1) / R : 0;
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto fold = [&](const float4 v, float m, float l) {
      const float top = fmaxf(M, m), f = M == top ? 1.0f : ex2(M - top), g = m == top ? 1.0f : ex2(m - top);
      M = top;
      L = L * f + l * g;
      acc.x = acc.x * f + v.x * g, acc.y = acc.y * f + v.y * g, acc.z = acc.z * f + v.z * g, acc.w = acc.w * f + v.w * g;
    };
    if (c0 < c1) {
      for (int cb = c0 + mine; cb <= c1; cb += 16) {
        float4 v[4];
        float rw[4], lw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float* p = part_of(min(cb + 4 * u, c1), s0);
          v[u] = *reinterpret_cast<const float4*>(p + w * 128 + 4 * lane);
          rw[u] = p[1024 + w];
          lw[u] = p[1032 + w];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (cb + 4 * u <= c1) fold(v[u], rw[u], lw[u]);
      }
    }
    quarter[warp][lane] = acc;
    if (lane == 0) qsum[warp] = make_float2(M, L);
    __syncthreads();
    // written by the streaming kernel where one CTA had the whole head; the last head's twin
    // of an odd count writes what the head itself writes
    if (mine || (nsb && c0 == c1)) return;
    for (int u = 1; u < 4; ++u) fold(quarter[warp + u][lane], qsum[warp + u].x, qsum[warp + u].y);
    const bool none = L == 0.f;
    const float r = none ? 0.f : 1.0f / L;
    __nv_bfloat16* dst = a.out + (static_cast<size_t>(b) * a.Hq + q) * 128 + 4 * lane;
    *reinterpret_cast<uint2*>(dst) = none ? make_uint2(0, 0) : make_uint2(pack_bf16(acc.x * r, acc.y * r), pack_bf16(acc.z * r, acc.w * r));
    if (none && nsb && lane == 0) set_err(a.err, kErrNoValidSlot);
    return;
  }
  const int s = (blockIdx.x - pairs) * 256 + threadIdx.x;
  if (static_cast<int>(blockIdx.x - pairs) * 256 >= nsb * 16) return;
  const bool mine = s < nsb * 16 && s < a.S;
  // eight threads per query head, the parts over them
  const int sub = threadIdx.x & 7;
  for (int q0 = 0; q0 < a.Hq; q0 += 32) {
    const int q = min(q0 + (static_cast<int>(threadIdx.x) >> 3), a.Hq - 1);
    const int h = q / group, w = q - h * group;
    const int s0 = first + h * nsb, c0 = s0 / R, c1 = (s0 + nsb - 1) / R;
    float M = -INFINITY, L = 0.f;
    if (c0 == c1) {
      const float2 v = *reinterpret_cast<const float2*>(a.stats + (static_cast<size_t>(b * Hkv + h) * 8 + w) * 2);
      if (sub == 0) M = v.x, L = v.y;
    } else {
      for (int c = c0 + sub; c <= c1; c += 8) {
        const float* p = part_of(c, s0);
        join(M, L, p[1024 + w], p[1032 + w]);
      }
    }
#pragma unroll
    for (int o = 4; o; o >>= 1)
      join(M, L, __shfl_xor_sync(0xffffffffu, M, o), __shfl_xor_sync(0xffffffffu, L, o));
    if (sub == 0) fin[q] = make_float2(M > -INFINITY ? M : 0.f, L == 0.f ? 0.f : 1.0f / L);
  }
  float* dst = a.step_score + static_cast<size_t>(b) * a.S + s;
  float top = mine ? *dst : 0.f;
  const float before = top;
  __syncthreads();
  if (!mine) return;
  bool nan = false;
  auto fold = [&](float x, int q) {
    const float2 f = fin[q];
    const float p = ex2(x - f.x) * f.y;
    nan |= p != p;
    top = fmaxf(top, p);
  };
  const float* x = a.logits + (static_cast<size_t>(b * Hkv) * a.s16 + s) * a.gs;
  const size_t head = static_cast<size_t>(a.s16) * a.gs;
#pragma unroll 4
  for (int h = 0; h < Hkv; ++h, x += head) {
    if (a.gs == 2) {
      const float2 v = *reinterpret_cast<const float2*>(x);
      fold(v.x, h * group);
      if (group > 1) fold(v.y, h * group + 1);
    } else {
      const float4 v = *reinterpret_cast<const float4*>(x);
      fold(v.x, h * group);
      fold(v.y, h * group + 1);
      fold(v.z, h * group + 2);
      if (group > 3) fold(v.w, h * group + 3);
      if (a.gs == 8) {
        const float4 u = *reinterpret_cast<const float4*>(x + 4);
        fold(u.x, h * group + 4);
        if (group > 5) fold(u.y, h * group + 5);
        if (group > 6) fold(u.z, h * group + 6);
        if (group > 7) fold(u.w, h * group + 7);
      }
    }
  }
  if (nan) set_err(a.err, kErrNanScore);
  if (top > before) *dst = top;
}

// Attention over short sequences in one launch: W warps of a CTA share a (sequence, kv head), so
// nothing is left to join between CTAs and the logits for the score stay in shared memory.
// Bound by latency: lengths, pages, one block's loads, two or three blocks of arithmetic a warp;
// blocks come straight into registers, the next one's loads in flight (W = 16 has no registers
// for that, and few blocks a warp).
constexpr int kShortBlocks = 128;      // blocks of a head at most (2048 slots)
constexpr int kShortSmem = 168 * 1024;
constexpr int kShortAlways = 16;          // blocks of a head up to which this form always wins
constexpr long long kShortTotal = 16384;  // beyond them: blocks of all heads at most
constexpr int kShortSpread = 148 * 16;    // warps that are resident at once

template <int W, bool kScore>
__global__ void __launch_bounds__(W > 8 ? 512 : 256, W > 8 ? 1 : 2) short_kernel(const AttnArgs a) {
  constexpr int kTeam = W > 8 ? 16 : 8, kHeads = kTeam / W;  // warps and heads of a CTA
  extern __shared__ __align__(16) float smem_f[];
  auto part = reinterpret_cast<float(*)[8][kHeadPitch]>(smem_f);  // [kTeam]
  float* logits = smem_f + kTeam * 8 * kHeadPitch;               // [kHeads][s16][gs]
  __shared__ float ref[kTeam][8], sum[kTeam][8];
  __shared__ float2 fin[kHeads][8];
  __shared__ Moves moves[kTeam];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int Hkv = a.pool.Hkv, group = a.Hq / Hkv, slot = warp / W, wi = warp % W;
  const int hid = blockIdx.x * kHeads + slot;
  const bool mine = hid < a.pool.B * Hkv;
  const int b = mine ? hid / Hkv : 0, h = mine ? hid - b * Hkv : 0;
  int n = mine ? a.lens[b] : 0;
  if (n < 0 || n > a.limit) {
    if (h == 0 && wi == 0 && lane == 0) set_err(a.err, kErrIndex);
    n = n < 0 ? 0 : a.limit;
  }
  const int nsb = (n + 15) >> 4, ppb = a.pool.page >> 4;
  float* lg = logits + static_cast<size_t>(slot) * a.s16 * a.gs;
  Sums sums;
  sums.clear(&moves[warp]);
  if (wi < nsb) {
    // pages of this warp's blocks wi, wi + W, ...: lane i the i-th
    const int my_blk = wi + W * lane;
    int page = -1;
    if (my_blk < nsb) page = a.pool.table[static_cast<size_t>(b) * a.pool.max_pages + my_blk / ppb];
    uint4 qf[4];
    const float unit = load_query(a.q + (static_cast<size_t>(b) * a.Hq + h * group + g) * 128, g < group, a.scale, t, qf);
    const float xs[2] = {__shfl_sync(0xffffffffu, unit, 8 * t), __shfl_sync(0xffffffffu, unit, 8 * t + 4)};
    auto q_of = [&](int j) { return qf[j]; };
    const bool ok_page = static_cast<unsigned>(page) < static_cast<unsigned>(a.pool.n_pages);
    if (my_blk < nsb && !ok_page) set_err(a.err, kErrIndex);
    const uint32_t oks = __ballot_sync(0xffffffffu, ok_page);
    const int sg = 4 * (g >> 1) + (g & 1);
    struct Raw {
      uint4 k0, k1, v0, v1, s0, s1;
      uint2 f0, f1;
      int pos;
    };
    auto fetch = [&](int i, Raw& r) {  // this warp's i-th block
      const int blk = wi + W * i, s = blk * 16 + (lane & 15);
      r.pos = s < n ? (a.slot_pos ? a.slot_pos[static_cast<size_t>(b) * a.S + s] : 0) : -1;
      const int pg = __shfl_sync(0xffffffffu, page, i);
      if (!(oks >> i & 1u)) {
        r = Raw{};
        r.pos = -1;
        return;
      }
      const uint8_t* p = a.pool.base + ((static_cast<size_t>(pg) * Hkv + h) * ppb + blk % ppb) * kBlock;
      r.k0 = *reinterpret_cast<const uint4*>(p + 64 * sg + 16 * t);
      r.k1 = *reinterpret_cast<const uint4*>(p + 64 * (sg + 2) + 16 * t);
      r.f0 = *reinterpret_cast<const uint2*>(p + kKScale + 8 * sg);
      r.f1 = *reinterpret_cast<const uint2*>(p + kKScale + 8 * (sg + 2));
      r.v0 = *reinterpret_cast<const uint4*>(p + 1024 + 64 * g + 16 * t);
      r.v1 = *reinterpret_cast<const uint4*>(p + 1536 + 64 * g + 16 * t);
      r.s0 = *reinterpret_cast<const uint4*>(p + kVScale + 32 * t);
      r.s1 = *reinterpret_cast<const uint4*>(p + kVScale + 32 * t + 16);
    };
    auto process = [&](const Raw& r, int blk) {
      const uint32_t mask = __ballot_sync(0xffffffffu, r.pos >= 0);  // both halves hold the 16 slots
      float x[4];
      block_logits(r.k0, r.k1, r.f0, r.f1, q_of, xs, x);
      mask_logits(x, mask >> sg);
      if (kScore && 2 * t < a.gs) {
        float* to = lg + (blk * 16 + sg) * a.gs + 2 * t;
        *reinterpret_cast<float2*>(to) = make_float2(x[0], x[1]);
        *reinterpret_cast<float2*>(to + 2 * a.gs) = make_float2(x[2], x[3]);
      }
      const uint4 s0 = mask_scales(r.s0, mask >> (4 * t)), s1 = mask_scales(r.s1, mask >> (4 * t + 2));
      float top[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
      uint4 u0 = s0, u1 = s1;
      if (sums.moved) u0 = sums.scaled(s0), u1 = sums.scaled(s1);
      if (sums.vote(top, or4(u0) | or4(u1), lane, [&](uint32_t (&m)[4]) {
            m[0] = max(max_half(s0.x), max_half(s1.x)), m[1] = max(max_half(s0.y), max_half(s1.y));
            m[2] = max(max_half(s0.z), max_half(s1.z)), m[3] = max(max_half(s0.w), max_half(s1.w));
          }))
        u0 = sums.scaled(s0), u1 = sums.scaled(s1);
      sums.weigh(x, r.v0, r.v1, u0, u1);
    };
    const int count = (nsb - wi + W - 1) / W;
    Raw cur;
    fetch(0, cur);
    for (int i = 0; i < count; ++i) {
      if (W <= 8) {
        Raw next;
        if (i + 1 < count) fetch(i + 1, next);
        process(cur, wi + W * i);
        cur = next;
      } else {
        process(cur, wi + W * i);
        if (i + 1 < count) fetch(i + 1, cur);
      }
    }
  }
  sums.leave(ref[warp], sum[warp], part[warp], group, wi < nsb, g, t);
  __syncthreads();
  for (int q = wi; q < group && mine; q += W) {  // one query head per warp, four dims per lane
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, ref[slot * W + w][q]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float rw = ref[slot * W + w][q], lw = sum[slot * W + w][q];
      if (rw > -INFINITY || lw != 0.f) {  // also a NaN sum
        const float fw = rw == M ? 1.0f : ex2(rw - M);
        const float4 v = *reinterpret_cast<const float4*>(&part[slot * W + w][q][4 * lane]);
        L += lw * fw;
        acc.x += v.x * fw, acc.y += v.y * fw, acc.z += v.z * fw, acc.w += v.w * fw;
      }
    }
    const bool none = L == 0.f;
    const float r = none ? 0.f : 1.0f / L;
    __nv_bfloat16* dst = a.out + (static_cast<size_t>(b) * a.Hq + h * group + q) * 128 + 4 * lane;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc.x * r, acc.y * r), pack_bf16(acc.z * r, acc.w * r));
    if (lane == 0) {
      fin[slot][q] = make_float2(M > -INFINITY ? M : 0.f, r);
      if (none && n > 0) set_err(a.err, kErrNoValidSlot);
    }
  }
  if (!kScore) return;
  __syncthreads();
  for (int s = wi * 32 + lane; s < nsb * 16 && s < a.S; s += W * 32) {
    float top = 0.f;
    bool nan = false;
    for (int q = 0; q < group; ++q) {
      const float2 f = fin[slot][q];
      const float p = ex2(lg[s * a.gs + q] - f.x) * f.y;
      nan |= p != p;
      top = fmaxf(top, p);
    }
    if (nan) set_err(a.err, kErrNanScore);
    // the kv heads' CTAs meet here; non-negative floats order like their bits
    if (top > 0.f) atomicMax(reinterpret_cast<int*>(a.step_score + static_cast<size_t>(b) * a.S + s), __float_as_int(top));
  }
}

static bool aligned16(const void* p) { return !misaligned(p, 16); }

static int floats_per_row(int group) { return group <= 2 ? 2 : group <= 4 ? 4 : 8; }

// Sequences per launch: their lengths fit shared memory and the line of blocks 32 bits.
static int seqs_per_launch(int B, int Hkv, int limit) {
  const long long line = static_cast<long long>(Hkv) * ((limit + 15) / 16);
  long long n = kMaxSeqs;
  if (line * n > 0x7fff0000ll) n = 0x7fff0000ll / line;
  return static_cast<int>(n < B ? n : B);
}

// Warps per head of the one-launch form, 0 where the streaming form is the faster one.
// Measured, one launch against streaming, without a score (28 heads over 4): 4.6 against 6.8 us
// at 64 kv heads of 64 slots, 35.2 against 57 at 2048 of 256 (so always up to 16 blocks), 10.3
// against 10.4 at 64 of 1024, 18.3 against 23.2 at 512 of 512, 16.0 against 18.9 at 128 of 2048;
// but 33.6 against 31.8 at 512 of 1024 and 32.9 against 27.8 at 256 of 2048.
static int short_warps(int B, int Hkv, int limit) {
  const long long heads = static_cast<long long>(B) * Hkv, nsb = (limit + 15) / 16;
  if (nsb > kShortAlways && (nsb > kShortBlocks || heads * nsb > kShortTotal)) return 0;
  if (heads > 0x7ffffff0ll) return 0;
  int W = 1;  // a lane keeps one block's page; all warps at once where there are few heads
  while (W < 16 && (32 * W < nsb || (W < nsb && heads * 2 * W <= kShortSpread))) W *= 2;
  return W;
}

static long long workspace_bytes(int B, int Hq, int Hkv, int limit, bool score) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || limit < 0 || short_warps(B, Hkv, limit)) return 0;
  long long n = kHeaderBytes + kPartBytes;
  if (score) {
    const long long pairs = static_cast<long long>(seqs_per_launch(B, Hkv, limit)) * Hkv;
    n += pairs * 64 + pairs * ((limit + 15ll) / 16 * 16) * floats_per_row((Hq + Hkv - 1) / Hkv) * 4;
  }
  return n;
}

static long long limit_of(const Pool& pool, bool bounded, int S) {  // slots of a sequence at most
  const long long n = static_cast<long long>(pool.max_pages) * pool.page;
  return bounded && S < n ? S : n;
}

template <int W>
static int launch_short(cudaStream_t stream, const AttnArgs& a) {
  constexpr int kTeam = W > 8 ? 16 : 8;
  auto kernel = a.step_score ? short_kernel<W, true> : short_kernel<W, false>;
  if (prepare_device(reinterpret_cast<const void*>(kernel), kShortSmem) <= 0)
    return fail(kStatusCuda, "kv4_attn: no usable CUDA device");
  const size_t smem = (kTeam * 8 * kHeadPitch + (a.step_score ? kTeam / W * a.s16 * a.gs : 0)) * sizeof(float);
  const int heads = a.pool.B * a.pool.Hkv, per = kTeam / W;
  const cudaError_t e = launch_pdl(kernel, dim3((heads + per - 1) / per), dim3(kTeam * 32), smem, stream, dim3(0), a);
  if (e != cudaSuccess) return fail(kStatusCuda, "kv4_attn launch: %s", cudaGetErrorString(e));
  return kStatusOk;
}

static int attend(cudaStream_t stream, int B, int Hq, const Pool& pool, const void* q, const int* lens,
                  const int* slot_pos, int S, float scale, void* out, float* step_score, void* ws, long long ws_bytes,
                  int* err) {
  if (const int W = short_warps(B, pool.Hkv, static_cast<int>(limit_of(pool, slot_pos || step_score, S)))) {
    AttnArgs a{};
    a.q = static_cast<const __nv_bfloat16*>(q);
    a.pool = pool;
    a.lens = lens;
    a.slot_pos = slot_pos;
    a.out = static_cast<__nv_bfloat16*>(out);
    a.step_score = step_score;
    a.err = err;
    a.scale = scale;
    a.Hq = Hq;
    a.S = S;
    a.limit = static_cast<int>(limit_of(pool, slot_pos || step_score, S));
    a.s16 = (a.limit + 15) / 16 * 16;
    a.gs = floats_per_row(Hq / pool.Hkv);
    switch (W) {
      case 1: return launch_short<1>(stream, a);
      case 2: return launch_short<2>(stream, a);
      case 4: return launch_short<4>(stream, a);
      case 8: return launch_short<8>(stream, a);
      default: return launch_short<16>(stream, a);
    }
  }
  if (!ws || !aligned16(ws)) return fail(kStatusArg, "kv4_attn: no aligned workspace");
  const int Hkv = pool.Hkv, group = Hq / Hkv;
  const long long limit = limit_of(pool, slot_pos || step_score, S);
  const int each = seqs_per_launch(B, Hkv, static_cast<int>(limit));
  if (each <= 0) return fail(kStatusUnsupported, "kv4_attn: too many heads and slots");
  if (ws_bytes < workspace_bytes(B, Hq, Hkv, static_cast<int>(limit), step_score != nullptr))
    return fail(kStatusArg, "kv4_attn: workspace of %lld bytes is too small", ws_bytes);
  auto kernel = step_score ? attend_kernel<true> : attend_kernel<false>;
  const int sms = prepare_device(reinterpret_cast<const void*>(kernel), sizeof(Smem));
  if (sms <= 0) return fail(kStatusCuda, "kv4_attn: no usable CUDA device");
  cudaError_t e;
  const int nsb = static_cast<int>((limit + 15) / 16);
  for (int b0 = 0; b0 < B; b0 += each) {
    AttnArgs a;
    a.q = static_cast<const __nv_bfloat16*>(q) + static_cast<size_t>(b0) * Hq * 128;
    a.pool = pool;
    a.pool.B = B - b0 < each ? B - b0 : each;
    a.pool.table = pool.table + static_cast<size_t>(b0) * pool.max_pages;
    a.lens = lens + b0;
    a.slot_pos = slot_pos ? slot_pos + static_cast<size_t>(b0) * S : nullptr;
    a.out = static_cast<__nv_bfloat16*>(out) + static_cast<size_t>(b0) * Hq * 128;
    a.step_score = step_score ? step_score + static_cast<size_t>(b0) * S : nullptr;
    uint8_t* w = static_cast<uint8_t*>(ws);
    a.header = reinterpret_cast<int*>(w);
    a.part = reinterpret_cast<float*>(w + kHeaderBytes);
    a.stats = step_score ? reinterpret_cast<float*>(w + kHeaderBytes + kPartBytes) : nullptr;
    a.logits = step_score ? a.stats + static_cast<size_t>(each) * Hkv * 16 : nullptr;
    a.err = err;
    a.scale = scale;
    a.Hq = Hq;
    a.S = S;
    a.limit = static_cast<int>(limit);
    a.s16 = nsb * 16;
    a.gs = floats_per_row(group);
    const long long line = static_cast<long long>(a.pool.B) * Hkv * nsb;
    const int least = nsb < kMinBlocks ? nsb : kMinBlocks;
    long long grid = (line + least - 1) / least;
    const int most = kCtas * sms < kMaxCtas ? kCtas * sms : kMaxCtas;
    grid = grid < 1 ? 1 : grid > most ? most : grid;
    e = launch_pdl(kernel, dim3(static_cast<unsigned>(grid)), dim3(kWarps * 32), sizeof(Smem), stream, dim3(0), a);
    if (e != cudaSuccess) return fail(kStatusCuda, "kv4_attn launch: %s", cudaGetErrorString(e));
    const int chunks = step_score ? (nsb * 16 + 255) / 256 : 0;
    e = launch_pdl(combine_kernel, dim3((Hq + 1) / 2 + chunks, a.pool.B), dim3(256), step_score ? Hq * sizeof(float2) : 0, stream,
                   dim3(0), a);
    if (e != cudaSuccess) return fail(kStatusCuda, "kv4_attn launch: %s", cudaGetErrorString(e));
  }
  return kStatusOk;
}

// From here on eight rows per CTA, below one.  One against eight, 28 + 2 * 4 heads: 6.5 us and 9.3
// at 512 rows, 11.3 and 14.3 at 1024, 19.3 and 15.9 at 2048, 40 and 17 at 4096; 32 + 2 * 8 heads
// with norms: 20 and 33 at 1024, 35 and 36 at 2048, 53 and 37 at 3000.  (Two rows per CTA would be
// the fastest from 768 to 2048: 6.9 us at 1024 rows, 10.9 at 2047.)
constexpr int kManyRows = 2048;

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
  if (!kv4::aligned16(q_out)) return fail(kvbp::kStatusArg, "kv4_append: q_out must be 16-byte aligned");
  if (Hq > 0 && kvbp::overlap(qkv, 2ll * ((rows - 1ll) * ldq + (Hq + 2ll * Hkv) * 128), q_out, 256ll * rows * Hq))
    return fail(kvbp::kStatusArg, "kv4_append: q_out must not overlap qkv");
  const kv4::AppendArgs a{static_cast<const __nv_bfloat16*>(qkv), static_cast<const __nv_bfloat16*>(bias),
                          static_cast<const __nv_bfloat16*>(q_norm_w), static_cast<const __nv_bfloat16*>(k_norm_w),
                          inv_freq, positions, slots, seq, p, static_cast<__nv_bfloat16*>(q_out), dev_err, ldq, rows,
                          rows_per_seq, Hq,
                          kv4::aligned16(qkv) && ldq % 8 == 0 && kv4::aligned16(bias) && kv4::aligned16(q_norm_w) && kv4::aligned16(k_norm_w), eps};
  const cudaError_t e =
      rows >= kv4::kManyRows
          ? kvbp::launch_pdl(kv4::append_kernel<8>, dim3((static_cast<unsigned>(rows) + 7) / 8), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), dim3(0), a)
          : kvbp::launch_pdl(kv4::append_kernel<1>, dim3(rows), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), dim3(0), a);
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
  if (row_stride < 128 || head_stride < 128 || row_stride % 8 || head_stride % 8 || !kv4::aligned16(k_out) ||
      !kv4::aligned16(v_out))
    return fail(kvbp::kStatusArg, "kv4_gather: output rows must be 128 apart or more and 16-byte aligned");
  if (Hkv > 65535) return fail(kvbp::kStatusArg, "kv4_gather: bad size");
  const cudaError_t e = kvbp::launch_pdl(
      kv4::gather_kernel, dim3((static_cast<unsigned>(rows) + 31) / 32, Hkv), dim3(256), 0,
      reinterpret_cast<cudaStream_t>(stream), dim3(0), slots, seq, rows_per_seq, rows, p,
      static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), static_cast<long long>(row_stride),
      static_cast<long long>(head_stride), dev_err);
  if (e != cudaSuccess) return fail(kvbp::kStatusCuda, "kv4_gather launch: %s", cudaGetErrorString(e));
  return kvbp::kStatusOk;
}

extern "C" int64_t kvbp_kv4_attn_workspace(int32_t B, int32_t Hq, int32_t Hkv, int32_t max_slots, int32_t with_score) {
  return kv4::workspace_bytes(B, Hq, Hkv, max_slots, with_score != 0);
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
  if (Hq > 4096) return fail(kvbp::kStatusUnsupported, "kv4_attn: %d query heads > 4096", Hq);
  if (S < 0 || ((slot_pos || step_score) && S == 0)) return fail(kvbp::kStatusArg, "kv4_attn: bad slot stride");
  if (!kv4::aligned16(q) || !kv4::aligned16(out))
    return fail(kvbp::kStatusArg, "kv4_attn: q and out must be 16-byte aligned");
  if (kvbp::overlap(q, 256ll * B * Hq, out, 256ll * B * Hq))
    return fail(kvbp::kStatusArg, "kv4_attn: out must not overlap q");
  return kv4::attend(reinterpret_cast<cudaStream_t>(stream), B, Hq, p, q, lens, slot_pos, S, scale, out, step_score,
                     workspace, workspace_bytes, dev_err);
}
