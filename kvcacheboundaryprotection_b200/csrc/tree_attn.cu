// Attention of a tree of drafted tokens over the slot cache on the 5th-generation tensor cores
// (tcgen05 + TMEM), with the eviction score of every (node, key).
//
//   out[b, t, h] = sum_s p_s v_s,  p = softmax(scale * q . k) over the live slots of sequence b and
//   the node's ancestors (itself among them);  score[b, t, key] = max over the heads of p.
//
// A kv head's rows are its G = Hq / Hkv query heads of every node: T * G rows read the same keys, so
// a cache tile is fetched once for all of them, and with more than a few rows the products belong on
// the tensor cores.  Rows are cut into row tiles of whole nodes (at most 128 rows = TMEM lanes).
// A unit is (sequence, kv head) with one row tile (form A), or with a pair of row tiles that share
// each key tile (form B, T * G > 128); its key tiles are the cache's and, last, the drafted nodes'.
// All units' key tiles stand in one line that is cut into equal ranges, one per CTA, whatever the
// lengths; a unit cut by a border leaves partial results (sum, running maximum, accumulator) that
// combine_kernel joins.
//
// attend_kernel, one CTA per SM (ranges over all SMs, or with few units a cluster of CTAs for each that
// joins its parts in shared memory):
//   * producer warp: K and V tiles (128 keys, 32 KiB each) by 3-D TMA through one ring in the order the
//     products need them; Q once per unit, rows of small trees 2 or 4 times over the TMEM lanes;
//   * MMA warp: item i = S_w = Q . K^T into TMEM (w = i & 1), then O_w += P . V with P read from TMEM;
//     form A: the items are the unit's key tiles in turn, two accumulators; form B: the two row tiles of
//     each key tile;
//   * softmax warps, a thread per row and part of the columns (copies of a row take a part each; a row
//     without copies has two warps, 16 in all): the tile's maximum, weights 2^(c s - c m) in bf16 packed
//     over S's columns, their sum.  The reference maximum m moves only when a row's maximum passes it by
//     more than 2^8 in weight (exact in fp32, and bf16 weights keep their 8 bits wherever they lie), so
//     that O is rescaled rarely;
//   * mask warp: the live bits of each key tile from slot_pos / lens; V rows of dead slots and
//     unused nodes are zeroed in shared memory before the product reads them (0 * NaN is NaN), and
//     drafted V elements that are not finite, which rows off their branch must not meet, are taken out
//     and added by the rows that see them.
// Rounding: S, sums and O are fp32; a weight is rounded once to bf16 (half a step, 2^-8 of it), in form A
// the sum that divides is that of the rounded weights (an error common to all cancels), in form B, where
// the issue slots count, that of the unrounded ones; out is rounded once.  The other attention kernels over
// bf16 caches hold the weights as a sum of two bf16.  Here that costs a second P . V product and a second conversion: 218 -> 241 us
// (64 sequences x 5 nodes x 4104 slots), 176 -> 225 (1 x 64 x 131071), 119-123 -> 126-130 (12 ragged x 33), 40.1 -> 41.8
// (16 x 16 x 1032), 19.0 -> 19.4 (1 x 8 x 256), and takes the error of out (2-norm, against 64 bits) from 0.0018-0.0022
// to the 0.0017 of its own rounding: a quarter of the time of large trees for less than a rounding of out.
// Measured on B200, calls on changing inputs: 64 sequences x 5 nodes x 4104 slots, 8 kv heads: 218 us, 4.7 TB/s of the
// 6.46 of a copy; 1 x 64 nodes x 131071 slots, 8 kv heads: 176 us, bound by the chain S -> weights -> P . V of each
// row tile.  Replayed from a graph on the same inputs, a part of which is then in L2, 187 and 143 us; in that
// state the first takes 122 us without the loads and 180 without the softmax (the two overlap but for the start of
// each unit), the second 128 without the weights' arithmetic, its tensor pipe 45 % busy.  Exponentials
// on the FMA pipe instead of the MUFU for 1/8 to 5/8 of the columns were slower (161 -> 166-180 us at the time).
//
// combine_kernel joins the parts of units that a border cut.  score_kernel forms p again from the final row
// statistics: S^T = K . Q^T with a slot per thread, so that the maximum over heads stays in the thread and
// the score rows are written along the slots (16 x 16 nodes x 1032 slots, 4 kv heads: 16 us of 37, replayed).
#include <type_traits>

#include "common.cuh"
#include "kvbp_internal.h"

namespace kvbp {
namespace ta {

constexpr int kD = 128;
constexpr int kMaxNodes = 128;
constexpr int kKeys = 128;
constexpr int kHalf = 128 * 128;  // a 64-column half of a [128][128] bf16 tile: 16 KiB
constexpr int kTile = 2 * kHalf;
// softmax warps: 8, or 16 where a row's columns are not already shared by its copies
constexpr int halves_of(int copies) { return copies == 1 ? 2 : 1; }
constexpr int threads_of(int copies) { return halves_of(copies) * 256 + 128; }
constexpr int kAhead = 8;  // barriers in turn over the key tiles: more than the ring holds of either kind
constexpr int kNf = 8;  // units' records of non-finite drafted values kept at a time
constexpr float kLog2e = 1.4426950408889634f;

// shared memory (from a 1024-aligned base): Q (32 KiB a row tile), the ring, then
constexpr int slots_of(int copies, bool form_b) { return form_b || copies > 1 ? 5 : 6; }
constexpr int kOffStat = 7 * kTile;                  // float4 [128]
constexpr int kOffBars = kOffStat + 128 * 16;        // mbarriers
constexpr int kOffMask = kOffBars + 384;             // uint4 [kAhead] live bits
constexpr int kOffNf = kOffMask + kAhead * 16;            // uint4 [kNf]
constexpr int kOffMisc = kOffNf + kNf * 16;          // TMEM address, flag, start of the range
constexpr int kSmem = kOffMisc + 64;
static_assert(kSmem <= 232448, "shared memory");

// What the two warps of the same 32 rows tell each other lies in two words a TMEM lane, maxima and sums alike.
// Nothing but their own barriers orders these uses (the pairs of warps drift apart by more than a unit), so
// each word belongs to one pair for good.
constexpr int pair_word(int half, int lane128) { return half * 128 + lane128; }
constexpr bool pair_words_apart() {
  for (int i = 0; i < 256; ++i)
    for (int k = 0; k < 256; ++k)
      if (i % 128 / 32 != k % 128 / 32 && pair_word(i / 128, i % 128) == pair_word(k / 128, k % 128)) return false;
  return true;
}
static_assert(pair_words_apart(), "a word of two pairs of warps");

struct Args {
  int B, T, Hq, Hkv, S, G;
  int npt;    // nodes of a row tile
  int pairs;  // units per (sequence, kv head)
  float c;    // |scale| * log2(e), > 0
  int neg;    // scale < 0
  int grid;
  int join;   // (Join) CTAs of the cluster that works on a unit and joins it itself
  __nv_bfloat16* out;
  const __nv_bfloat16* vd;
  const int *parents, *slot_pos, *lens;
  float* part;     // [grid][2][128][rows] partial accumulators, rows = 128 (form A) or 256
  float2* pstat;   // [grid][2][rows] their maximum and sum(s)
  float* lse;      // [B][T][Hq] log2 of the sum of weights, for the score (or null)
  int* base;       // [B + 1] first key tile of each sequence (with lens)
  int* err;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- pairs of fp32 in one register pair (two results per issue slot)
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// maximum of three, NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Barrier of 64 threads; true in all where it is in one.
__device__ __forceinline__ bool any_of_pair(int id, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred.aligned q, %2, 64, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(v)), "r"(id)
      : "memory");
  return r != 0;
}

// log2 of a row's sum of weights; NaN where all its logits are -inf, as its outputs are (0 / 0); infinite, so that
// every weight is 0, where the node is unused.
__device__ __forceinline__ float lse_of(float M, float L, float c, bool used) {
  if (!used) return __int_as_float(0x7f800000);
  return L == 0.f ? __int_as_float(0x7fffffff) : fmaf(M, c, log2f(L));
}

// Key tiles of sequence b: its cache's, and the drafted one.
__device__ __forceinline__ int len_of(const Args& a, int b) {
  if (!a.lens) return a.S;
  const int n = a.lens[b];
  return n < 0 ? 0 : n > a.S ? a.S : n;
}
__device__ __forceinline__ int tiles_of(int len) { return (len + kKeys - 1) / kKeys + 1; }

// The nodes that node t sees (bits), none where it is unused.
__device__ __forceinline__ bool node_sees(const int* par, int t, uint32_t (&sees)[4], int* err) {
  sees[0] = sees[1] = sees[2] = sees[3] = 0;
  for (;;) {
    const int p = par[t];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((t >> 5) == i) sees[i] |= 1u << (t & 31);
    if (p >= t || p < -1) {
      if (p >= t) set_err(err, kErrIndex);
      sees[0] = sees[1] = sees[2] = sees[3] = 0;
      return false;
    }
    if (p < 0) return true;
    t = p;
  }
}

// A value that is the same in every lane, so that the compiler knows it and keeps what follows from it
// in uniform registers (the operands of tcgen05 and TMA instructions).
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// The parents of a tree, four to a lane, and the same walk with them: a whole warp, each lane from its
// node ``t`` (-1: none).  Steps cost a few shuffles; through memory they were 0.3 us each.
struct Parents {
  int p[4];
  __device__ __forceinline__ void load(const int* par, int T, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = i * 32 + lane < T ? par[i * 32 + lane] : -2;
  }
  __device__ __forceinline__ bool sees(int t, int T, uint32_t (&bits)[4]) const {
    bits[0] = bits[1] = bits[2] = bits[3] = 0;
    bool used = t >= 0;
    while (__any_sync(0xffffffffu, t >= 0)) {
      int up = __shfl_sync(0xffffffffu, p[0], t & 31);
      if (T > 32) {
#pragma unroll
        for (int i = 1; i < 4; ++i) {
          const int v = __shfl_sync(0xffffffffu, p[i], t & 31);
          if ((t >> 5) == i) up = v;
        }
      }
      if (t >= 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((t >> 5) == i) bits[i] |= 1u << (t & 31);
        if (up >= t || up < -1) used = false;
        t = used ? up : -1;
      }
    }
    if (!used) bits[0] = bits[1] = bits[2] = bits[3] = 0;
    return used;
  }
};

// A walk over the CTA's range of key tiles, unit by unit, by whole warps.
struct Walk {
  int t, end;        // global key tiles left: [t, end)
  int b, base, len;  // sequence, its first tile, its length
  int h, pair, tile0, n, nt;  // unit, first key tile of the segment, their number, tiles of the unit
  int seg;
  __device__ __forceinline__ void start(int t0, int t1, int b0, int base0) {
    t = t0, end = t1, b = b0, base = base0, n = 0, seg = -1;
  }
  __device__ __forceinline__ bool next(const Args& a) {
    t += n;
    if (t >= end) return false;
    const int per_head = a.pairs;
    len = uniform(len_of(a, b));
    nt = tiles_of(len);
    while (t - base >= nt * a.Hkv * per_head) {
      base += nt * a.Hkv * per_head;
      ++b;
      len = uniform(len_of(a, b));
      nt = tiles_of(len);
    }
    const int rel = t - base, u = rel / nt;
    tile0 = rel - u * nt;
    h = u / per_head;
    pair = u - h * per_head;
    n = min(nt - tile0, end - t);
    ++seg;
    return true;
  }
  __device__ __forceinline__ bool whole() const { return n == nt; }
};

template <int F, bool FormB, bool Score, bool Join>
__global__ void __launch_bounds__(threads_of(F), 1)
    attend_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap kdmap,
                  const __grid_constant__ CUtensorMap vdmap, const Args a) {
  extern __shared__ __align__(1024) uint8_t base[];
  constexpr int NS = slots_of(F, FormB);
  constexpr int kRowsF = 128 / F;  // TMEM lanes of one copy of the rows
  constexpr int H = halves_of(F);  // warps that share a row's columns
  constexpr int kProducer = 8 * H, kMma = kProducer + 1, kMask = kProducer + 2;  // one more fills the warpgroup
  constexpr int NQ = FormB ? 2 : 1;
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + kOffBars);
  uint64_t* kfull = bars;          // [kAhead] K landed
  uint64_t* vfull = bars + 8;      // [kAhead] V landed
  uint64_t* vok = bars + 16;       // [kAhead] the mask warp has cleaned the V tile
  uint64_t* empty = bars + 24;     // [NS] ring slot: its product is done
  uint64_t* sfull = bars + 30;     // [2] S written
  uint64_t* pready = bars + 32;    // [2] P written (4 H warps)
  uint64_t* odone = bars + 36;     // the unit's last products are done
  uint64_t* qfull = bars + 38;
  uint64_t* qfree = bars + 39;
  uint64_t* drain = bars + 40;     // after a wait that gave up
  float4* stat = reinterpret_cast<float4*>(base + kOffStat);
  uint4* masks = reinterpret_cast<uint4*>(base + kOffMask);
  uint4* nfs = reinterpret_cast<uint4*>(base + kOffNf);
  uint32_t* misc = reinterpret_cast<uint32_t*>(base + kOffMisc);
  volatile int* bad = reinterpret_cast<volatile int*>(misc + 1);
  uint8_t* ring = base + NQ * kTile;
  float* joint = reinterpret_cast<float*>(ring + NS * kTile);  // F > 1: [2][128 lanes][32 dims]
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < 41; ++i) mbar_init(bars + i, i == 32 || i == 33 ? 4 * H : 1);
    *bad = 0;
    if (smem_u32(base) & 1023) {  // the swizzle needs the base aligned
      *bad = 1;
      set_err(a.err, kErrWaitTimeout);
    }
    fence_barrier_init();
  }
  if (warp == kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(misc)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  pdl_launch_dependents();
  pdl_wait();
  // the range of key tiles, and the sequence that it starts in
  if (warp == kProducer) {
    const int per = a.Hkv * a.pairs;
    int total, b0, base0;
    // border c of the CTAs' ranges, total * c / g over g CTAs (no more than there are tiles)
    auto border = [&](int c) {
      const int g = min(a.grid, total), q = total / g;
      return c < g ? q * c + (total - q * g) * c / g : total;
    };
    if (!a.lens) {
      const int nt = tiles_of(a.S) * per;
      total = nt * a.B;
      const int t0 = border(blockIdx.x);
      b0 = t0 / nt;
      base0 = b0 * nt;
    } else {
      total = 0;
      for (int i = 0; i < a.B; i += 32) {
        int v = i + lane < a.B ? tiles_of(len_of(a, i + lane)) * per : 0;
        if (i + lane < a.B && blockIdx.x == 0 && (a.lens[i + lane] < 0 || a.lens[i + lane] > a.S))
          set_err(a.err, kErrIndex);
        int incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += x;
        }
        if (blockIdx.x == 0 && i + lane < a.B) a.base[i + lane] = total + incl - v;
        total += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (blockIdx.x == 0 && lane == 0) a.base[a.B] = total;
      const int t0 = border(blockIdx.x);
      b0 = base0 = 0;
      int run = 0;
      for (int i = 0; i < a.B; i += 32) {
        int v = i + lane < a.B ? tiles_of(len_of(a, i + lane)) * per : 0;
        int incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += x;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, i + lane < a.B && run + incl - v <= t0);
        if (hit) {
          const int l = 31 - __clz(hit);
          b0 = i + l;
          base0 = run + __shfl_sync(0xffffffffu, incl - v, l);
        }
        run += __shfl_sync(0xffffffffu, incl, 31);
        if (run > t0) break;
      }
    }
    if (lane == 0) {
      misc[2] = border(blockIdx.x);
      misc[3] = border(blockIdx.x + 1);
      misc[4] = b0;
      misc[5] = base0;
    }
  }
  tc_before();
  __syncthreads();
  tc_after();
  constexpr uint32_t tmem = 0;  // all 512 columns: they begin at 0
  if (tid == 0 && misc[0] != tmem) {
    *bad = 1;
    set_err(a.err, kErrWaitTimeout);
  }
  Walk w;
  w.start(uniform(misc[2]), uniform(misc[3]), uniform(misc[4]), uniform(misc[5]));
  const int n_tiles = w.end - w.t;
  const int R = a.npt * a.G;

  // A wait gives up after a while (or at once when another one has): the walk then runs to its end
  // without touching data, so that every barrier of threads is still met.
  auto wait = [&](uint64_t* bar, uint32_t ph) {
    if (mbar_try_wait(bar, ph)) return;
    for (uint32_t i = 0; i < (1u << 22); ++i) {
      if (mbar_try_wait(bar, ph)) return;
      if (*bad) return;
      if (i > 1024) __nanosleep(32);
    }
    set_err(a.err, kErrWaitTimeout);
    *bad = 1;
  };
  // ring position of the K / V tile of the CTA's j-th key tile
  auto k_pos = [&](int j) { return FormB ? 2 * j : j ? 2 * j - 1 : 0; };
  auto v_pos = [&](int j) { return FormB ? 2 * j + 1 : j + 1 < n_tiles ? 2 * j + 2 : 2 * j + 1; };

  // the softmax threads hold their part of a row of S: registers move to them from the other warps
  // (640 threads at 96 = 512 at 104 + 128 at 64)
  if (warp >= kProducer) {
    if constexpr (H == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (warp == kProducer) {
    // ================================ TMA ==============================================
    const bool leader = elect_one();
    if (leader) {
      prefetch_tmap(&qmap);
      prefetch_tmap(&kmap);
      prefetch_tmap(&vmap);
    }
    int k_issued = 0, v_issued = 0, q_issued = 0;
    auto load = [&](const Walk& x, int tile, bool value, int j) {
      const int pos = value ? v_pos(j) : k_pos(j), s = pos % NS;
      if (pos >= NS) wait(&empty[s], (pos / NS - 1) & 1);
      (value ? v_issued : k_issued) = j + 1;
      const bool drafted = tile == x.nt - 1;
      const CUtensorMap* m = drafted ? (value ? &vdmap : &kdmap) : (value ? &vmap : &kmap);
      const int y = drafted ? 0 : tile * kKeys, z = x.b * a.Hkv + x.h;
      uint64_t* bar = (value ? vfull : kfull) + j % kAhead;
      if (leader && !*bad) {
        mbar_expect_tx(bar, kTile);
        tma_load_3d(ring + s * kTile, m, bar, 0, y, z);
        tma_load_3d(ring + s * kTile + kHalf, m, bar, 64, y, z);
      }
    };
    Walk last = w;  // the unit and tile whose V is still to be loaded
    int last_tile = -1, j = 0;
    while (w.next(a)) {
      if (w.seg > 0) wait(qfree, (w.seg - 1) & 1);
      q_issued = w.seg + 1;
      if (leader && !*bad) {
        mbar_expect_tx(qfull, NQ * F * 2 * R * 128);
        for (int r = 0; r < NQ * F; ++r)
          for (int hf = 0; hf < 2; ++hf)
            tma_load_3d(base + (FormB ? r * kTile : r * kRowsF * 128) + hf * kHalf, &qmap, qfull, 64 * hf, w.h * a.G,
                        w.b * a.T + (FormB ? w.pair * 2 + r : 0) * a.npt);
      }
      for (int i = 0; i < w.n; ++i, ++j) {
        load(w, w.tile0 + i, false, j);
        if (FormB) {
          load(w, w.tile0 + i, true, j);
        } else {
          if (j > 0) load(last, last_tile, true, j - 1);
          last = w;
          last_tile = w.tile0 + i;
        }
      }
    }
    if (!FormB && j > 0) load(last, last_tile, true, j - 1);
    if (leader && *bad) {  // a wait has given up: the copies in flight land before the shared memory goes
      for (int k = max(0, k_issued - NS); k < k_issued; ++k)
        mbar_wait_bounded(&kfull[k % kAhead], (k / kAhead) & 1, 1u << 14);
      for (int k = max(0, v_issued - NS); k < v_issued; ++k)
        mbar_wait_bounded(&vfull[k % kAhead], (k / kAhead) & 1, 1u << 14);
      if (q_issued) mbar_wait_bounded(qfull, (q_issued - 1) & 1, 1u << 14);
    }
    __syncwarp();
  } else if (warp == kMma) {
    // ================================ tensor cores =====================================
    // (the warp walks together, so that everything but the issue itself is in uniform registers: one
    // lane walking alone spent 2200 cycles on an item's 16 products, 1000 of them useful)
    const bool leader = elect_one();
    constexpr uint32_t idS = tc_idesc(128, 128, 0), idO = tc_idesc(128, 128, 1);
    const uint64_t dq = tc_sdesc(smem_u32(base)), dk = tc_sdesc(smem_u32(ring)), dv = tc_sdesc(smem_u32(ring), kHalf, 1024);
    // One commit an item: S(i + 2) is issued after P V(i), so that its completion says that both are done,
    // and the softmax warps that wait for it anyway hand Q, K and V back.  (A commit costs 115 cycles of
    // this warp, a wait that is over 100: at five waits and three commits an item they were half its time.)
    auto issue_s = [&](int i, int j) {  // S of item i (key tile j of the CTA) into S_w
      const int x = i & 1, s = k_pos(j) % NS;
      if (!FormB || x == 0) wait(&kfull[j % kAhead], (j / kAhead) & 1);
      tc_after();
      const uint64_t q = dq + (FormB ? x * (kTile >> 4) : 0), k = dk + s * (kTile >> 4);
      if (leader) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const uint32_t off = ((ks >> 2) * kHalf + (ks & 3) * 32) >> 4;
          tc_mma(tmem + x * 128, q + off, k + off, idS, ks > 0);
        }
        tc_commit(&sfull[x]);
      }
      __syncwarp();
    };
    auto issue_pv = [&](int i, int j, bool first, bool last) {
      const int x = i & 1, s = v_pos(j) % NS;
      wait(&pready[x], (i >> 1) & 1);  // (its warps have waited for the cleaned V)
      tc_after();
      const uint64_t v = dv + s * (kTile >> 4);
      if (leader) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          tc_mma_ts(tmem + 256 + x * 128, tmem + x * 128 + ks * 8, v + ks * (16 * 128 >> 4), idO, !first || ks > 0);
        if (last) tc_commit(odone);
      }
      __syncwarp();
    };
    // the S products run two items ahead of the P V products, over unit borders too
    Walk ahead = w;
    int ai = 0, aj = 0, left = 0, aw = 0;  // next S item, its key tile, tiles left in its unit, row tile
    auto s_next = [&]() {
      if (left == 0) {
        if (!ahead.next(a)) return;
        left = ahead.n;
        aw = 0;
        wait(qfull, ahead.seg & 1);
      }
      if (FormB) {
        issue_s(ai, aj);
        if (aw == 1) ++aj, --left;
        aw ^= 1;
      } else {
        issue_s(ai, aj);
        ++aj, --left;
      }
      ++ai;
    };
    s_next();
    s_next();
    int i = 0, j = 0;
    while (w.next(a)) {
      const int items = FormB ? 2 * w.n : w.n;
      for (int k = 0; k < items; ++k, ++i) {
        issue_pv(i, j, k < 2, k == items - 1);
        if (!FormB || (k & 1)) ++j;
        s_next();
      }
    }
    if (leader && *bad) {  // products in flight end before TMEM goes
      tc_commit(drain);
      mbar_wait_bounded(drain, 0, 1u << 14);
    }
    __syncwarp();
  } else if (warp == kMask) {
    // ================================ masks ============================================
    int j = 0;
    auto value = [&](const Walk& x, int tile, int j) {
      const int s = v_pos(j) % NS;
      const bool drafted = tile == x.nt - 1;
      uint32_t m[4];
      if (drafted) {
        Parents tree;
        tree.load(a.parents + static_cast<size_t>(x.b) * a.T, a.T, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t sees[4];
          const int t = i * 32 + lane;
          m[i] = 0;
          if (i * 32 < a.T) {
            m[i] = __ballot_sync(0xffffffffu, tree.sees(t < a.T ? t : -1, a.T, sees));
            if (t < a.T && tree.p[i] >= t) set_err(a.err, kErrIndex);
          }
        }
      } else {
        int p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int sl = tile * kKeys + i * 32 + lane;
          p[i] = sl < x.len ? (a.slot_pos ? a.slot_pos[static_cast<size_t>(x.b) * a.S + sl] : 0) : -1;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) m[i] = __ballot_sync(0xffffffffu, p[i] >= 0);
      }
      wait(&vfull[j % kAhead], (j / kAhead) & 1);
      uint8_t* v = ring + s * kTile;
      if ((m[0] & m[1] & m[2] & m[3]) != 0xffffffffu) {
        // 16 lanes a row: its two 128-byte halves
        const int off = ((lane >> 3) & 1) * kHalf + (lane & 7) * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t dead = ~m[i];
          if (lane >= 16) dead >>= 16;
          for (int r = 0; r < 16; ++r)
            if ((dead >> r) & 1u)
              *reinterpret_cast<uint4*>(v + (i * 32 + (lane & 16) + r) * 128 + off) = make_uint4(0, 0, 0, 0);
        }
      }
      if (drafted) {
        // elements that are not finite (exponent all ones) leave the product; nf: their nodes
        uint32_t nf[4] = {0, 0, 0, 0};
        __syncwarp();
        const int off = ((lane >> 3) & 1) * kHalf + (lane & 7) * 16;
        for (int r = 0; r < a.T; r += 2) {
          const int row = r + (lane >> 4);
          uint32_t hit = 0;
          if (row < a.T) {
            uint4* at = reinterpret_cast<uint4*>(v + row * 128 + off);
            uint4 x4 = *at;
            uint32_t* wd = reinterpret_cast<uint32_t*>(&x4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if ((wd[i] & 0x7F80u) == 0x7F80u) wd[i] &= 0xFFFF0000u, hit = 1;
              if ((wd[i] & 0x7F800000u) == 0x7F800000u) wd[i] &= 0xFFFFu, hit = 1;
            }
            if (hit) *at = x4;
          }
          const uint32_t vote = __ballot_sync(0xffffffffu, hit);
          if (vote & 0xffffu) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if ((r >> 5) == i) nf[i] |= 1u << (r & 31);
          }
          if (vote >> 16) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (((r + 1) >> 5) == i) nf[i] |= 1u << ((r + 1) & 31);
          }
        }
        if (lane == 0) nfs[x.seg % kNf] = make_uint4(nf[0], nf[1], nf[2], nf[3]);
      }
      if (lane == 0) masks[j % kAhead] = make_uint4(m[0], m[1], m[2], m[3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&vok[j % kAhead]);
    };
    while (w.next(a))
      for (int i = 0; i < w.n; ++i, ++j) value(w, w.tile0 + i, j);
  }
  } else {
    // ================================ softmax ==========================================
    if constexpr (H == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    constexpr int NC = kRowsF / H;  // columns of a tile that a thread takes
    // accumulator (items i with i & 1 == x), part of the columns, TMEM lanes
    const int x = warp / (4 * H), hc = H == 2 ? (warp >> 2) & 1 : 0, quarter = warp & 3;
    const int row = F == 4 ? lane : F == 2 ? (quarter & 1) * 32 + lane : quarter * 32 + lane;
    const int copy = F == 4 ? quarter : F == 2 ? quarter >> 1 : 0;
    const int pair_bar = 6 + x * 4 + quarter;  // (H == 2) the two warps of the same rows
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS = tmem + x * 128 + lanes, tO = tmem + 256 + x * 128 + lanes;
    const bool idle = F == 1 && quarter * 32 >= R;  // no row of this warp is in use
    const float NEG_INF = -__int_as_float(0x7f800000);
    const float c = a.c;
    const uint64_t c2 = pack2(c, c);
    float* xchg = reinterpret_cast<float*>(stat) + x * 256;  // (H == 2) pair_word
    const int at = quarter * 32 + lane;  // this thread's TMEM lane
    const int word0 = pair_word(0, at), word1 = pair_word(1, at);
    const bool releases = quarter == 0 && hc == 0 && (!FormB || x == 1);  // hands tiles back
    int i0 = 0, j0 = 0;  // the CTA's items and key tiles before this unit
    int done = 0;        // items of this accumulator so far
    Parents tree;
    int tree_of = -1;  // the sequence whose tree it is
    while (w.next(a)) {
      const int rt = FormB ? w.pair * 2 + x : 0;  // row tile
      const int node = rt * a.npt + row / a.G;
      const bool in = row < R && node < a.T;
      const bool has_draft = w.tile0 + w.n == w.nt;
      uint32_t own[NC / 32];  // the drafted nodes of this thread's columns that the row sees
#pragma unroll
      for (int q = 0; q < NC / 32; ++q) own[q] = 0;
      bool used = false;
      {
        if (w.b != tree_of) {
          tree.load(a.parents + static_cast<size_t>(w.b) * a.T, a.T, lane);
          tree_of = w.b;
        }
        uint32_t sees[4];
        used = tree.sees(in ? node : -1, a.T, sees);
        if constexpr (F == 4) {
          own[0] = copy == 0 ? sees[0] : copy == 1 ? sees[1] : copy == 2 ? sees[2] : sees[3];
        } else {
          const bool upper = F == 2 ? copy == 1 : hc == 1;
          own[0] = upper ? sees[2] : sees[0], own[1] = upper ? sees[3] : sees[1];
        }
      }
      float m = NEG_INF, l = 0.f, lx = 0.f;
      const int items = FormB ? 2 * w.n : w.n;
      const int first = (i0 & 1) == x ? 0 : 1;
      for (int k = first; k < items; k += 2) {
        const int kt = FormB ? k >> 1 : k, j = j0 + kt;
        wait(&sfull[x], done & 1);
        if (releases) {  // products up to this S are done
          if (lane == 0) {
            mbar_arrive(&empty[k_pos(j) % NS]);
            if (k >= 2) mbar_arrive(&empty[v_pos(FormB ? j - 1 : j - 2) % NS]);
            if (k == items - 1) mbar_arrive(qfree);
          }
          __syncwarp();
        }
        wait(&vok[j % kAhead], (j / kAhead) & 1);
        tc_after();
        if (!idle) {
          uint32_t s[NC];
#pragma unroll
          for (int q = 0; q < NC / 32; ++q)
            tc_ld32_raw(tS + (copy * H + hc) * NC + q * 32, *reinterpret_cast<uint32_t(*)[32]>(s + q * 32));
          tc_wait_ld();
          uint32_t mw[NC / 32];
          if (has_draft && kt == w.n - 1) {
#pragma unroll
            for (int q = 0; q < NC / 32; ++q) mw[q] = own[q];
          } else {
            const uint32_t* mk = reinterpret_cast<const uint32_t*>(masks + j % kAhead) + (copy * H + hc) * (NC / 32);
#pragma unroll
            for (int q = 0; q < NC / 32; ++q) mw[q] = mk[q];
          }
          if (a.neg) {
#pragma unroll
            for (int e = 0; e < NC; ++e) s[e] ^= 0x80000000u;
          }
          uint32_t all = mw[0];
#pragma unroll
          for (int q = 1; q < NC / 32; ++q) all &= mw[q];
          if (!__all_sync(0xffffffffu, all == 0xffffffffu)) {
#pragma unroll
            for (int e = 0; e < NC; ++e) s[e] = ((mw[e / 32] >> (e % 32)) & 1u) ? s[e] : 0xff800000u;
          }
          float top[4] = {__uint_as_float(s[0]), __uint_as_float(s[1]), __uint_as_float(s[2]), __uint_as_float(s[3])};
#pragma unroll
          for (int e = 4; e < NC - 4; e += 8)
#pragma unroll
            for (int q = 0; q < 4; ++q) top[q] = max3(top[q], __uint_as_float(s[e + q]), __uint_as_float(s[e + 4 + q]));
          top[0] = max3(top[0], __uint_as_float(s[NC - 4]), __uint_as_float(s[NC - 3]));
          top[1] = max3(top[1], __uint_as_float(s[NC - 2]), __uint_as_float(s[NC - 1]));
          float tm = max3(max3(top[0], top[1], top[2]), top[3], top[3]);
          // (a NaN moves the reference to NaN: the row ends as NaN)
          auto moves = [&]() { return in && !(tm <= m) && !((tm - m) * c <= 8.f); };
          // the two warps of a row move together.  Past this barrier both have read S, whose columns
          // P will take.
          const bool any = H == 2 ? any_of_pair(pair_bar, moves()) : __any_sync(0xffffffffu, moves());
          if (any) {
            if (H == 2) {
              xchg[hc ? word1 : word0] = tm;
              named_bar(pair_bar, 64);
              tm = max3(tm, xchg[hc ? word0 : word1], tm);
            }
            const bool move = moves();
            const float f = move ? (m == NEG_INF ? 0.f : ex2((m - tm) * c)) : 1.f;
            if (move) m = tm;
            l *= f;
            lx *= f;
            if (k >= 2) {  // (S of this item was issued after the previous P V product: that is done)
#pragma unroll 1
              for (int q = hc * (8 / H); q < (hc + 1) * (8 / H); ++q) {
                uint32_t o[16];
                tc_ld16_raw(tO + q * 16, o);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tc_st16(tO + q * 16, o);
              }
              tc_wait_st();
            }
            if (H == 2) {  // either half of P lets a product begin: O is whole before that
              tc_before();
              named_bar(pair_bar, 64);
            }
          }
          const float mc = (m == NEG_INF ? 0.f : m) * c;
          const uint64_t nmc2 = pack2(-mc, -mc);
          uint64_t add[2] = {0, 0}, addx[2] = {0, 0};
          // the weights, packed over the same registers
#pragma unroll
          for (int e = 0; e < NC; e += 2) {
            float p0, p1;
            unpack2(fma2(pack2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, nmc2), p0, p1);
            p0 = ex2(p0), p1 = ex2(p1);
            uint32_t pk;
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(pk) : "f"(p1), "f"(p0));
            if (FormB || Score) addx[e / 2 % 2] = add2(addx[e / 2 % 2], pack2(p0, p1));
            if (!FormB)
              add[e / 2 % 2] =
                  add2(add[e / 2 % 2], pack2(__uint_as_float(pk << 16), __uint_as_float(pk & 0xFFFF0000u)));
            s[e / 2] = pk;
          }
          if constexpr (F == 1) {
            tc_st32(tS + hc * 32, *reinterpret_cast<uint32_t(*)[32]>(s));
          } else {
            // this copy's columns, zeros in the others'
            uint32_t zero[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) zero[e] = 0;
#pragma unroll
            for (int q = 0; q < F; ++q) {
              if (q == copy) {
                if constexpr (F == 4)
                  tc_st16(tS + q * 16, *reinterpret_cast<uint32_t(*)[16]>(s));
                else
                  tc_st32(tS + q * 32, *reinterpret_cast<uint32_t(*)[32]>(s));
              } else {
                tc_st16(tS + q * (64 / F), zero);
                if constexpr (F == 2) tc_st16(tS + q * 32 + 16, zero);
              }
            }
          }
          tc_wait_st();
          float a0, a1, b0, b1;
          if (FormB || Score) {
            unpack2(addx[0], a0, a1);
            unpack2(addx[1], b0, b1);
            lx += (a0 + a1) + (b0 + b1);
          }
          if (!FormB) {
            unpack2(add[0], a0, a1);
            unpack2(add[1], b0, b1);
            l += (a0 + a1) + (b0 + b1);
          }
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pready[x]);
        ++done;
      }
      i0 += items;
      j0 += w.n;
      if (FormB) l = lx;
      // ---- the unit's rows: accumulators in TMEM, statistics in the threads
      wait(odone, w.seg & 1);
      if (releases && lane == 0 && first < items) mbar_arrive(&empty[v_pos(j0 - (FormB || ((items - 1 - first) & 1) == 0 ? 1 : 2)) % NS]);
      float f0 = 1.f, f1 = 0.f, M = m, L = l, Lx = lx;
      if (H == 2) {  // the sums of the two warps of a row
        if (hc == 1) xchg[word0] = l, xchg[word1] = lx;
        named_bar(pair_bar, 64);
        if (hc == 0) {
          L = l = l + xchg[word0];
          Lx = lx = lx + xchg[word1];
          if (FormB) xchg[word0] = l, xchg[word1] = lx;
        }
        if (FormB) {
          named_bar(pair_bar, 64);
          if (hc == 1) L = xchg[word0], Lx = xchg[word1];
          named_bar(pair_bar, 64);  // read before this pair writes them again in the next unit
        } else {
          named_bar(3, 256 * H);
        }
      }
      if (!FormB) {
        // the two accumulators of a row lie in the same TMEM lane: both warpgroups join them, each
        // for half the dims
        if (x == 1 && hc == 0) stat[at] = make_float4(m, l, lx, 0.f);
        named_bar(1, 256 * H);
        float m0 = m, m1 = m;
        if (x == 0 && hc == 0) {
          const float4 o = stat[at];
          m1 = o.x;
          M = fmaxf(m, m1);
          const float e0 = m == NEG_INF ? 0.f : ex2((m - M) * c), e1 = m1 == NEG_INF ? 0.f : ex2((m1 - M) * c);
          L = e0 * l + e1 * o.y;
          Lx = e0 * lx + e1 * o.z;
          // (the threads that know one of m0, m1 need the other: it is not the larger, M, or both are)
          stat[at] = make_float4(fminf(m, m1), M, L, Lx);
        }
        named_bar(2, 256 * H);
        if (x == 1 || hc == 1) {
          const float4 o = stat[at];
          M = o.y, L = o.z, Lx = o.w;
          const float other = m == M ? o.x : M;
          (x == 0 ? m1 : m0) = other;
        }
        f0 = m0 == NEG_INF ? 0.f : ex2((m0 - M) * c);
        f1 = m1 == NEG_INF ? 0.f : ex2((m1 - M) * c);
        if (M != M || L != L) f0 = f1 = 1.f;  // a NaN logit: L is NaN, the row will be
        if (F > 1) {
          // and the copies of the row, each with the sums of its own columns
          const float mine = M;
          float Mf = NEG_INF, Lf = 0.f, Lxf = 0.f;
#pragma unroll
          for (int q = 0; q < F; ++q) Mf = fmaxf(Mf, stat[q * kRowsF + row].y);
#pragma unroll
          for (int q = 0; q < F; ++q) {
            const float4 o = stat[q * kRowsF + row];
            const float e = o.y == NEG_INF ? 0.f : ex2((o.y - Mf) * c);
            Lf = fmaf(e, o.z, Lf);
            Lxf = fmaf(e, o.w, Lxf);
          }
          const float e = mine == NEG_INF ? 0.f : ex2((mine - Mf) * c);
          f0 *= e, f1 *= e;
          M = Mf, L = Lf, Lx = Lxf;
        }
      }
      tc_after();
      const size_t orow = (static_cast<size_t>(w.b) * a.T + node) * a.Hq + static_cast<size_t>(w.h) * a.G + row % a.G;
      const bool whole = w.whole();
      const int rows = FormB ? 256 : 128;
      const int prow = FormB ? x * 128 + row : row;
      const size_t slot = static_cast<size_t>(blockIdx.x) * 2 + (w.seg > 0 ? 1 : 0);
      // (a dim's rows side by side: stores of whole lines.  A cluster's parts stay in shared memory: the
      // ring is idle once the CTA's one segment is done.)
      float* part = (Join ? reinterpret_cast<float*>(ring) : a.part + slot * kD * rows) + prow;
      float2* pstat = Join ? reinterpret_cast<float2*>(ring + kD * rows * 4) : a.pstat + slot * rows;
      float* pexact = Join ? reinterpret_cast<float*>(ring + kD * rows * 4 + rows * 8)
                           : reinterpret_cast<float*>(a.pstat + static_cast<size_t>(a.grid) * 2 * rows) + slot * rows;
      const bool ok = !*bad;
      if (in && ok && (FormB || x == 0) && copy == 0 && hc == 0) {
        if (!whole) {
          pstat[prow] = used ? make_float2(M, L) : make_float2(NEG_INF, -1.f);  // (-1: an unused node's)
          if (Score) pexact[prow] = Lx;
        } else if (Score) {
          a.lse[orow] = lse_of(M, Lx, c, used);
        }
      }
      const float inv = whole ? 1.f / L : 1.f;
      const uint4 nf4 = has_draft ? nfs[w.seg % kNf] : make_uint4(0, 0, 0, 0);
      bool odd = false;
      uint32_t sees[4] = {0, 0, 0, 0};
      if (nf4.x | nf4.y | nf4.z | nf4.w) {
        if (in) node_sees(a.parents + static_cast<size_t>(w.b) * a.T, node, sees, nullptr);
        odd = ((nf4.x & sees[0]) | (nf4.y & sees[1]) | (nf4.z & sees[2]) | (nf4.w & sees[3])) != 0;
      }
      // N finished sums of dims d0 .. of this thread's row go out
      auto put = [&](auto& o, int d0) {
        constexpr int N = sizeof(o) / 4;
        if (odd) {
          for (int t = 0; t < a.T; ++t) {
            const uint32_t nw = t < 32 ? nf4.x & sees[0] : t < 64 ? nf4.y & sees[1] : t < 96 ? nf4.z & sees[2] : nf4.w & sees[3];
            if (!((nw >> (t & 31)) & 1u)) continue;
            const __nv_bfloat16* v = a.vd + ((static_cast<size_t>(w.b) * a.Hkv + w.h) * a.T + t) * kD + d0;
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const float y = __bfloat162float(v[e]);
              if (!(fabsf(y) <= 3.4e38f)) o[e] += y;
            }
          }
        }
        if (!in || !ok) return;
        if (whole) {
          uint4* dst = reinterpret_cast<uint4*>(a.out + orow * kD + d0);
#pragma unroll
          for (int e = 0; e < N / 8; ++e) {
            uint32_t pk[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) pk[z] = used ? pack_bf16(o[e * 8 + 2 * z], o[e * 8 + 2 * z + 1]) : 0u;
            dst[e] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) part[static_cast<size_t>(d0 + e) * rows] = o[e];
        }
      };
      // 32 dims of the joined accumulators of this lane
      auto get = [&](float (&o)[32], int d0) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t r0[16], r1[16];
          tc_ld16_raw(tmem + 256 + lanes + d0 + q * 16, r0);
          tc_ld16_raw(tmem + 384 + lanes + d0 + q * 16, r1);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float v0 = f0 > 0.f ? __uint_as_float(r0[e]) * f0 : 0.f;
            const float v1 = f1 > 0.f ? __uint_as_float(r1[e]) * f1 : 0.f;
            o[q * 16 + e] = (v0 + v1) * inv;
          }
        }
      };
      if constexpr (FormB) {
        if (!idle && ok) {
#pragma unroll 1
          for (int q = hc * 2; q < hc * 2 + 2; ++q) {
            uint32_t r0[32];
            float o[32];
            tc_ld32_raw(tO + q * 32, r0);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(r0[e]) * inv;
            put(o, q * 32);
          }
        }
      } else if constexpr (F == 1) {
        if (!idle && ok) {
          float o[32];
          get(o, x * 64 + hc * 32);
          put(o, x * 64 + hc * 32);
        }
      } else {
        // the copies' sums meet in shared memory, 32 dims of each warpgroup's half at a time
        float* mine = joint + x * 128 * 32;
#pragma unroll 1
        for (int q = 0; q < 2; ++q) {
          if (ok) {
            float o[32];
            get(o, x * 64 + q * 32);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<float4*>(mine + at * 32 + ((e ^ (at & 7)) << 2)) =
                  make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
          named_bar(4 + x, 128);
          if (ok) {
            float o[32 / F];
#pragma unroll
            for (int e = 0; e < 8 / F; ++e) {
              float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
              for (int g = 0; g < F; ++g) {
                const int lg = g * kRowsF + row;
                const float4 v = *reinterpret_cast<float4*>(mine + lg * 32 + (((copy * (8 / F) + e) ^ (lg & 7)) << 2));
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
              }
              o[4 * e] = sum.x, o[4 * e + 1] = sum.y, o[4 * e + 2] = sum.z, o[4 * e + 3] = sum.w;
            }
            put(o, x * 64 + q * 32 + copy * (32 / F));
          }
          named_bar(4 + x, 128);
        }
      }
      tc_before();
      // both halves of a row are read before either accumulator is written again (and the statistics)
      if (!FormB) named_bar(3, 256 * H);
    }
  }
  __syncwarp();
  tc_before();
  __syncthreads();
  if (warp == kMma) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(misc[0]), "r"(512));
  if constexpr (Join) {
    // ---- the cluster's CTAs have the parts of one unit in their shared memory: each joins some of the
    // dims, eight at a time (a warp for 32 rows)
    cluster_sync_all();
    const int p = a.join, rank = blockIdx.x % p, u = blockIdx.x / p;
    const int b = u / (a.Hkv * a.pairs), h = u / a.pairs % a.Hkv, pair = u % a.pairs;
    constexpr int rows = FormB ? 256 : 128;
    const float NEG_INF = -__int_as_float(0x7f800000);
    const uint32_t mem = smem_u32(ring);
    const int d_lo = rank * 16 / p, d_hi = (rank + 1) * 16 / p;  // groups of 8 dims
    const int groups = (R + 31) / 32, units = groups * NQ * (d_hi - d_lo);
    if (warp < kProducer)
      for (int i = warp; i < units; i += kProducer) {
        const int d0 = (d_lo + i / (groups * NQ)) * 8, half = NQ == 2 ? i / groups % NQ : 0;
        const int r = i % groups * 32 + lane, t = (pair * NQ + half) * a.npt + r / a.G;
        if (r >= R || t >= a.T) continue;
        const int prow = half * 128 + r;
        float M = NEG_INF, L = 0.f, Lx = 0.f, o[8];
        float2 st[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q < p) st[q] = ld_dsmem_f2(mapa_u32(mem + kD * rows * 4 + prow * 8, q));
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q < p) M = fmaxf(M, st[q].x);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (q >= p) break;
          const uint32_t at = mapa_u32(mem + (d0 * rows + prow) * 4, q);
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = ld_dsmem_f32(at + e * rows * 4);
          const float f = st[q].x == NEG_INF ? 0.f : ex2((st[q].x - M) * a.c);
          L = fmaf(f, st[q].y, L);
          if (Score && d0 == 0) Lx = fmaf(f, ld_dsmem_f32(mapa_u32(mem + kD * rows * 4 + rows * 8 + prow * 4, q)), Lx);
          if (f != 0.f) {
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = fmaf(f, v[e], o[e]);
          }
        }
        const bool used = !(st[0].y < 0.f);
        const float inv = 1.f / L;
        const size_t orow = (static_cast<size_t>(b) * a.T + t) * a.Hq + static_cast<size_t>(h) * a.G + r % a.G;
        uint32_t pk[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) pk[e] = used ? pack_bf16(o[2 * e] * inv, o[2 * e + 1] * inv) : 0u;
        *reinterpret_cast<uint4*>(a.out + orow * kD + d0) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        if (Score && d0 == 0) a.lse[orow] = lse_of(M, Lx, a.c, used);
      }
    __syncwarp();
    cluster_sync_all();  // its parts are read before a CTA leaves
  }
}

// Joins the parts of units that a border cut: a block for 32 rows of a row tile (a lane each) and 32
// dims, four to a warp.
template <bool FormB, bool Score>
__global__ void __launch_bounds__(256) combine_kernel(const Args a) {
  pdl_launch_dependents();
  pdl_wait();
  const int warp = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  // blocks: sequence, kv head, pair, (row tile of the pair, 32 rows of it)
  const int groups = (a.npt * a.G + 31) / 32, per_unit = (FormB ? 2 : 1) * groups, per = a.Hkv * a.pairs;
  const int b = blockIdx.x / (per * per_unit), u = blockIdx.x / per_unit % per, part = blockIdx.x % per_unit;
  const int half = FormB ? part / groups : 0, r = part % groups * 32 + lane;
  const int h = u / a.pairs, rt = FormB ? u % a.pairs * 2 + half : 0;
  const int nt = tiles_of(len_of(a, b));
  const long long total = a.lens ? a.base[a.B] : static_cast<long long>(nt) * per * a.B;
  const long long t0 = (a.lens ? a.base[b] : static_cast<long long>(nt) * per * b) + static_cast<long long>(u) * nt;
  const long long g = total < a.grid ? total : a.grid;
  const int c0 = static_cast<int>(((t0 + 1) * g - 1) / total);
  const int c1 = static_cast<int>(((t0 + nt) * g - 1) / total);
  if (c0 == c1) return;  // written by the CTA that had it all
  const int t = rt * a.npt + r / a.G;
  if (r >= a.npt * a.G || t >= a.T) return;
  const int rows = FormB ? 256 : 128;
  const int prow = half * 128 + r;
  // the unit's first part is its CTA's second where it does not begin there
  const int later = total * c0 / g < t0 ? 1 : 0;
  auto slot = [&](int c) { return static_cast<size_t>(c) * 2 + (c == c0 ? later : 0); };
  const float NEG_INF = -__int_as_float(0x7f800000);
  float M = NEG_INF;
#pragma unroll 4
  for (int c = c0; c <= c1; ++c) M = fmaxf(M, a.pstat[slot(c) * rows + prow].x);
  const float* exact = reinterpret_cast<const float*>(a.pstat + static_cast<size_t>(a.grid) * 2 * rows);
  float L = 0.f, Lx = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int c = c0; c <= c1; ++c) {
    const size_t s = slot(c);
    const float2 st = a.pstat[s * rows + prow];
    const float* v = a.part + (s * kD + warp * 4) * rows + prow;
    const float v0 = v[0], v1 = v[rows], v2 = v[2 * rows], v3 = v[3 * rows];
    const float e = st.x == NEG_INF ? 0.f : ex2((st.x - M) * a.c);
    L = fmaf(e, st.y, L);
    if (Score && warp == 0) Lx = fmaf(e, exact[s * rows + prow], Lx);
    if (e != 0.f) o[0] = fmaf(e, v0, o[0]), o[1] = fmaf(e, v1, o[1]), o[2] = fmaf(e, v2, o[2]), o[3] = fmaf(e, v3, o[3]);
  }
  const bool used = !(a.pstat[slot(c0) * rows + prow].y < 0.f);
  const float inv = 1.f / L;
  const size_t orow = (static_cast<size_t>(b) * a.T + t) * a.Hq + static_cast<size_t>(h) * a.G + r % a.G;
  *reinterpret_cast<uint2*>(a.out + orow * kD + warp * 4) =
      used ? make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)) : make_uint2(0, 0);
  if (Score && warp == 0) a.lse[orow] = lse_of(M, Lx, a.c, used);
}

// ------------------------------------------------------------------------------------
// score: S^T = K . Q^T, a slot per TMEM lane, the columns query head by query head (nodes side by side),
// so that the maximum over the heads stays in the thread's registers and, over the kv heads, in its
// words of shared memory; the CTA max-accumulates it into the score at the end, along the slots.
// Several small CTAs share an SM: the loads of one hide behind the weights of another.
// ------------------------------------------------------------------------------------
constexpr int kScoreThreads = 9 * 32;  // 8 warps over the columns, one for TMA and MMA
constexpr int kScOffQ = kTile;                      // K, then Q of one item
constexpr int kScOffLse = 2 * kTile;                // float [128]
constexpr int kScOffSee = kScOffLse + 128 * 4;      // uint4 [128]
constexpr int kScOffBars = kScOffSee + kMaxNodes * 16;
constexpr int kScOffNan = kScOffBars + 64;          // uint32 [4] nodes with a NaN among their sums of weights
constexpr int kScOffMax = kScOffNan + 16;           // float [nodes, a multiple of 8][128 slots]
constexpr int score_smem(int T) { return kScOffMax + (T + 7) / 8 * 8 * 128 * 4; }

struct ScoreArgs {
  Args a;
  float* score;  // [B][T][S + T]
  int tiles;     // key tiles of a sequence: ceil(S / 128) + 1
  int hsplit;    // groups of kv heads
  int chunk;     // nodes of an item, a multiple of 8
  int gb;        // query heads of an item: gb * chunk <= 128
};

__global__ void __launch_bounds__(kScoreThreads, 3)
    score_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap kdmap, const ScoreArgs p) {
  extern __shared__ __align__(1024) uint8_t base[];
  const Args& a = p.a;
  float* best = reinterpret_cast<float*>(base + kScOffMax);
  float* slse = reinterpret_cast<float*>(base + kScOffLse);
  uint4* see = reinterpret_cast<uint4*>(base + kScOffSee);
  uint32_t* nans = reinterpret_cast<uint32_t*>(base + kScOffNan);
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + kScOffBars);
  uint64_t* full = bars;       // K and Q landed
  uint64_t* sfull = bars + 1;  // S^T written
  uint64_t* sfree = bars + 2;  // S^T read by the 8 warps
  uint64_t* drain = bars + 3;  // after a wait that gave up
  uint32_t* misc = reinterpret_cast<uint32_t*>(bars + 4);
  volatile int* bad = reinterpret_cast<volatile int*>(misc + 1);
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  const int tile = blockIdx.x, hg = blockIdx.y, b = blockIdx.z;
  const bool drafted = tile == p.tiles - 1;
  const int h0 = hg * a.Hkv / p.hsplit, h1 = (hg + 1) * a.Hkv / p.hsplit;
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(bars + i, i == 2 ? 8 : 1);
    *bad = 0;
    if (smem_u32(base) & 1023) {
      *bad = 1;
      set_err(a.err, kErrWaitTimeout);
    }
    fence_barrier_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(misc)), "r"(128));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  const int T8 = (a.T + 7) / 8 * 8;
  if (tid < 4) nans[tid] = 0;
  for (int i = tid; i < T8 * 128; i += kScoreThreads) best[i] = 0.f;
  pdl_launch_dependents();
  pdl_wait();
  if (drafted)
    for (int t = tid; t < a.T; t += kScoreThreads) {
      uint32_t s[4];
      node_sees(a.parents + static_cast<size_t>(b) * a.T, t, s, nullptr);
      see[t] = make_uint4(s[0], s[1], s[2], s[3]);
    }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = misc[0];
  const int len = len_of(a, b);
  const bool any = drafted || tile * kKeys < len;
  const int gparts = (a.G + p.gb - 1) / p.gb, chunks = (a.T + p.chunk - 1) / p.chunk;
  const int items = any ? (h1 - h0) * gparts * chunks : 0;
  // item i: kv head, first query head, first node (the kv head changes last: K is loaded once for it)
  auto head_of = [&](int i) { return h0 + i / (gparts * chunks); };
  auto g_of = [&](int i) { return i / chunks % gparts * p.gb; };
  auto node_of = [&](int i) { return i % chunks * p.chunk; };
  auto wait = [&](uint64_t* bar, uint32_t ph) {
    if (mbar_try_wait(bar, ph)) return;
    for (uint32_t i = 0; i < (1u << 22); ++i) {
      if (mbar_try_wait(bar, ph)) return;
      if (*bad) return;
      if (i > 1024) __nanosleep(32);
    }
    set_err(a.err, kErrWaitTimeout);
    *bad = 1;
  };
  if (warp == 8) {
    const bool leader = elect_one();
    int loaded = 0;
    auto load = [&](int i) {
      const int h = head_of(i), g0 = g_of(i), gn = min(p.gb, a.G - g0);
      const bool new_k = i == 0 || head_of(i - 1) != h;
      loaded = i + 1;
      if (!leader || *bad) return;
      mbar_expect_tx(full, (new_k ? kTile : 0) + gn * p.chunk * 256);
      for (int hf = 0; hf < 2; ++hf) {
        if (new_k) {
          if (drafted)
            tma_load_3d(base + hf * kHalf, &kdmap, full, 64 * hf, 0, b * a.Hkv + h);
          else
            tma_load_3d(base + hf * kHalf, &kmap, full, 64 * hf, tile * kKeys, b * a.Hkv + h);
        }
        for (int g = 0; g < gn; ++g)  // a query head's nodes: whole swizzle atoms of 8 rows
          tma_load_3d(base + kScOffQ + hf * kHalf + g * p.chunk * 128, &qmap, full, 64 * hf, h * a.G + g0 + g,
                      b * a.T + node_of(i));
      }
    };
    if (items > 0) load(0);
    const uint64_t dk = tc_sdesc(smem_u32(base)), dq = tc_sdesc(smem_u32(base + kScOffQ));
    for (int i = 0; i < items; ++i) {
      wait(full, i & 1);
      if (i > 0) wait(sfree, (i - 1) & 1);
      tc_after();
      const uint32_t id = tc_idesc(128, (min(p.gb, a.G - g_of(i)) * p.chunk + 15) / 16 * 16, 0);
      if (leader && !*bad) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const uint32_t off = ((ks >> 2) * kHalf + (ks & 3) * 32) >> 4;
          tc_mma(tmem, dk + off, dq + off, id, ks > 0);
        }
        tc_commit(sfull);
      }
      __syncwarp();
      if (i + 1 < items) {
        wait(sfull, i & 1);  // the product has read the buffers
        load(i + 1);
      }
    }
    if (leader && *bad) {  // copies and products in flight end before their memory goes
      tc_commit(drain);
      mbar_wait_bounded(drain, 0, 1u << 14);
      if (loaded) mbar_wait_bounded(full, (loaded - 1) & 1, 1u << 14);
    }
    __syncwarp();
  } else {
    const int sl = (warp & 3) * 32 + lane, part = warp >> 2;  // slot; which of every two blocks of 8 nodes
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int key = tile * kKeys + sl;
    const bool live = drafted ? sl < a.T
                              : key < len && (!a.slot_pos || a.slot_pos[static_cast<size_t>(b) * a.S + key] >= 0);
    for (int i = 0; i < items; ++i) {
      const int h = head_of(i), g0 = g_of(i), gn = min(p.gb, a.G - g0), n0 = node_of(i);
      named_bar(1, 256);  // the previous item's statistics have been read
      for (int r = tid; r < gn * p.chunk; r += 256) {
        const int t = n0 + r % p.chunk;
        const float l = t < a.T ? a.lse[(static_cast<size_t>(b) * a.T + t) * a.Hq + static_cast<size_t>(h) * a.G + g0 + r / p.chunk]
                                : __int_as_float(0x7f800000);
        slse[r] = l;
        if (l != l) atomicOr(&nans[t >> 5], 1u << (t & 31));
      }
      wait(sfull, i & 1);
      named_bar(2, 256);
      tc_after();
      for (int n = part * 8; n < p.chunk && n0 + n < a.T; n += 16) {
        float mx[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) mx[e] = 0.f;
        for (int g = 0; g < gn; g += 4) {
          uint32_t v[4][8];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (g + q < gn) tc_ld8_raw(tmem + lanes + (g + q) * p.chunk + n, v[q]);
          tc_wait_ld();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (g + q >= gn) break;
            const float4* ls = reinterpret_cast<const float4*>(slse + (g + q) * p.chunk + n);
            const float4 l0 = ls[0], l1 = ls[1];
            const float lse[8] = {l0.x, l0.y, l0.z, l0.w, l1.x, l1.y, l1.z, l1.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float s = __uint_as_float(v[q][e]);
              mx[e] = fmaxf(mx[e], ex2(fmaf(a.neg ? -s : s, a.c, -lse[e])));
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float* at = best + (n0 + n + e) * 128 + sl;
          *at = fmaxf(*at, mx[e]);
        }
      }
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sfree);
    }
    // (the blocks of nodes shift between warps from chunk to chunk: wait for all)
    named_bar(1, 256);
    if (live && any && !*bad) {
      for (int t = part; t < a.T; t += 2) {
        if (drafted) {
          const uint4 m = see[t];
          const uint32_t w = sl < 32 ? m.x : sl < 64 ? m.y : sl < 96 ? m.z : m.w;
          if (!((w >> (sl & 31)) & 1u)) continue;
        }
        // (a NaN logit makes all of the node's weights NaN; the maxima above leave NaN out)
        const bool nan = (nans[t >> 5] >> (t & 31)) & 1u;
        const float v = nan ? __int_as_float(0x7fffffff) : best[t * 128 + sl];
        if (nan) set_err(a.err, kErrNanScore);
        if (nan || v > 0.f)
          atomicMax(reinterpret_cast<int*>(p.score + (static_cast<size_t>(b) * a.T + t) * (static_cast<size_t>(a.S) + a.T) +
                                           (drafted ? a.S : tile * kKeys) + sl),
                    __float_as_int(v));
      }
    }
  }
  __syncwarp();
  tc_before();
  __syncthreads();
  if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(128));
}

}  // namespace ta

// ------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------
namespace {

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<EncodeFn>(ptr);
  }();
  return fn;
}

// [d2][d1][128] bf16 rows, boxes of 64 columns x b1 x b2
int map_rows(CUtensorMap* m, const void* ptr, long long d1, long long d2, int b1, int b2) {
  EncodeFn enc = encode_fn();
  if (!enc) return fail(kStatusCuda, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(d1), static_cast<cuuint64_t>(d2)};
  cuuint64_t strides[2] = {256, static_cast<cuuint64_t>(d1) * 256};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(b1), static_cast<cuuint32_t>(b2)};
  cuuint32_t one[3] = {1, 1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(kStatusCuda, "tree_attn: tensor map failed (%d)", static_cast<int>(r));
  return kStatusOk;
}

struct Plan {
  int form_b, npt, pairs, rows;
};

// Row tiles of whole nodes, at most 128 rows each: one (form A), or an even number of equal ones.
Plan plan_of(int T, int G) {
  const int cap = 128 / G;
  Plan p;
  p.form_b = T > cap;
  const int tiles = p.form_b ? 2 * ((T + 2 * cap - 1) / (2 * cap)) : 1;
  p.npt = (T + tiles - 1) / tiles;
  p.pairs = p.form_b ? tiles / 2 : 1;
  p.rows = p.form_b ? 256 : 128;
  return p;
}

constexpr int kMaxGrid = 148;  // workspace is sized for a whole B200

struct Work {
  long long part, pstat, lse, base, bytes;
};
Work work_of(int B, int T, int Hq, const Plan& p) {
  auto up = [](long long x) { return (x + 255) / 256 * 256; };
  Work w;
  w.part = 0;
  w.pstat = up(w.part + 2LL * kMaxGrid * p.rows * 512);
  w.lse = up(w.pstat + 2LL * kMaxGrid * p.rows * 12);
  w.base = up(w.lse + static_cast<long long>(B) * T * Hq * 4);
  w.bytes = up(w.base + (static_cast<long long>(B) + 1) * 4);
  return w;
}

}  // namespace
}  // namespace kvbp

#include "../../include/kvbp.h"

extern "C" int64_t kvbp_tree_attn_workspace(int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t S,
                                            int32_t with_score) {
  (void)S, (void)with_score;
  if (B <= 0 || T <= 0 || T > kvbp::ta::kMaxNodes || Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > 128) return 0;
  return kvbp::work_of(B, T, Hq, kvbp::plan_of(T, Hq / Hkv)).bytes;
}

extern "C" int kvbp_tree_attn(kvbp_stream_t stream, int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t head_dim,
                              int32_t S, const void* q, const void* kcache, const void* vcache, const void* k_draft,
                              const void* v_draft, const int32_t* parents, const int32_t* slot_pos,
                              const int32_t* lens, float scale, void* out, float* node_score, void* workspace,
                              int64_t workspace_bytes, int32_t* dev_err) {
  using namespace kvbp;
  using namespace kvbp::ta;
  if (!q || !k_draft || !v_draft || !parents || !out || (S > 0 && (!kcache || !vcache)))
    return fail(kStatusArg, "tree_attn: null pointer");
  if (head_dim != kD) return fail(kStatusUnsupported, "tree_attn: head_dim %d unsupported (only 128)", head_dim);
  if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || S < 0 || B > 65535) return fail(kStatusArg, "tree_attn: bad size");
  if (T <= 0 || T > kMaxNodes) return fail(kStatusUnsupported, "tree_attn: %d nodes (1 to %d)", T, kMaxNodes);
  const int G = Hq / Hkv;
  if (G > 128) return fail(kStatusUnsupported, "tree_attn: %d query heads per kv head (at most 128)", G);
  if (!(scale == scale) || scale - scale != 0.f) return fail(kStatusArg, "tree_attn: scale is not finite");
  if (misaligned(q, 16) || misaligned(kcache, 16) || misaligned(vcache, 16) || misaligned(k_draft, 16) ||
      misaligned(v_draft, 16) || misaligned(out, 16) || misaligned(workspace, 16))
    return fail(kStatusArg, "tree_attn: q, caches, drafts, out and workspace must be 16-byte aligned");
  const Plan p = plan_of(T, G);
  const long long tiles = (static_cast<long long>(S) + kKeys - 1) / kKeys + 1;
  const long long total = tiles * B * Hkv * p.pairs;
  if (total > 0x7fffffffLL || static_cast<long long>(B) * Hkv > 0x7fffffffLL ||
      static_cast<long long>(B) * T * Hq > 0x7fffffffLL || S > 0x7fffffff - 1024)
    return fail(kStatusArg, "tree_attn: too many keys or rows for one call");
  const Work wk = work_of(B, T, Hq, p);
  if (!workspace || workspace_bytes < wk.bytes)
    return fail(kStatusArg, "tree_attn: a workspace of %lld bytes is needed", wk.bytes);
  const long long nq = static_cast<long long>(B) * T * Hq * 256, nc = static_cast<long long>(B) * Hkv * S * 256,
                  nd = static_cast<long long>(B) * Hkv * T * 256,
                  ns = node_score ? static_cast<long long>(B) * T * (static_cast<long long>(S) + T) * 4 : 0;
  const struct {
    const void* p;
    long long n;
  } in[] = {{q, nq}, {kcache, nc}, {vcache, nc}, {k_draft, nd}, {v_draft, nd}, {parents, 4LL * B * T},
            {slot_pos, slot_pos ? 4LL * B * S : 0}, {lens, lens ? 4LL * B : 0}},
    written[] = {{out, nq}, {node_score, ns}, {workspace, wk.bytes}};
  for (int i = 0; i < 3; ++i) {
    for (const auto& r : in)
      if (r.n && written[i].n && overlap(written[i].p, written[i].n, r.p, r.n))
        return fail(kStatusArg, "tree_attn: an output or the workspace overlaps an input");
    for (int k = 0; k < i; ++k)
      if (written[i].n && written[k].n && overlap(written[i].p, written[i].n, written[k].p, written[k].n))
        return fail(kStatusArg, "tree_attn: out, node_score and workspace overlap");
  }
  CUtensorMap qm, km, vm, kdm, vdm;
  int st;
  if ((st = map_rows(&qm, q, Hq, static_cast<long long>(B) * T, G, p.npt))) return st;
  if ((st = map_rows(&kdm, k_draft, T, static_cast<long long>(B) * Hkv, kKeys, 1))) return st;
  if ((st = map_rows(&vdm, v_draft, T, static_cast<long long>(B) * Hkv, kKeys, 1))) return st;
  km = kdm, vm = vdm;  // never read without a cache
  if (S > 0) {
    if ((st = map_rows(&km, kcache, S, static_cast<long long>(B) * Hkv, kKeys, 1))) return st;
    if ((st = map_rows(&vm, vcache, S, static_cast<long long>(B) * Hkv, kKeys, 1))) return st;
  }
  const bool score = node_score != nullptr;
  const int copies = p.form_b ? 1 : p.npt * G <= 32 ? 4 : p.npt * G <= 64 ? 2 : 1;
  const int sms = prepare_device(reinterpret_cast<const void*>(attend_kernel<1, false, false, false>), kSmem);
  if (!sms) return fail(kStatusCuda, "tree_attn: no usable device");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Args a{};
  a.B = B, a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.S = S, a.G = G;
  a.npt = p.npt, a.pairs = p.pairs;
  a.neg = scale < 0.f;
  a.c = fmaxf(fabsf(scale) * kLog2e, 1e-30f);
  const int most = sms < kMaxGrid ? sms : kMaxGrid;
  a.grid = static_cast<int>(total < most ? total : most);
  a.join = 0;
  bool cut = true;  // some unit may lie in two CTAs' ranges
  if (!lens) {
    // How the units are shared out, by the time of the slowest CTA in key tiles:
    //  * equal ranges over all SMs: the best balance, but a CTA begins twice where a border lies inside a
    //    unit (about two), and a second launch joins the parts (about five);
    //  * n CTAs for each unit: borders between units;
    //  * the n a cluster, which joins its parts in shared memory (about one and a half), or n = 1.
    // Each wave of CTAs begins anew (about three).  clusters[n]: how many clusters of n CTAs with this much
    // shared memory a B200 holds.  On B200 (replayed): 64 units of 10 tiles 25 us by ranges over 148 CTAs, 20 us in
    // clusters of 2; 48 units of 65 (form B) 75 us by ranges, 70 us on 3 CTAs a unit; 512 units of 34
    // 189 us by ranges, 222 us in clusters of 2.
    static const int clusters[9] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
    const long long units = total / tiles, n_all = most / units;
    double best = static_cast<double>(total) / most + 10;
    if (n_all >= 1 && n_all <= tiles && (tiles + n_all - 1) / n_all + 8 < best) {
      best = static_cast<double>((tiles + n_all - 1) / n_all + 8);
      a.grid = static_cast<int>(units * n_all);
    }
    for (int n = 1; n <= 8 && n <= tiles; ++n) {
      const double waves = static_cast<double>((units + clusters[n] - 1) / clusters[n]);
      const double time = waves * ((tiles + n - 1) / n + 3) + (n > 1 ? 1.5 : 0);
      if (time < best) {
        best = time;
        cut = false;
        a.join = n;
        a.grid = static_cast<int>(units * n);
      }
    }
  }
  a.out = static_cast<__nv_bfloat16*>(out);
  a.vd = static_cast<const __nv_bfloat16*>(v_draft);
  a.parents = parents, a.slot_pos = S > 0 ? slot_pos : nullptr, a.lens = lens;
  a.part = reinterpret_cast<float*>(ws + wk.part);
  a.pstat = reinterpret_cast<float2*>(ws + wk.pstat);
  a.lse = reinterpret_cast<float*>(ws + wk.lse);
  a.base = reinterpret_cast<int*>(ws + wk.base);
  a.err = dev_err;
  cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  const bool joined = a.join > 1;
  auto pick = [&](auto score_c, auto join_c) {
    constexpr bool sc = decltype(score_c)::value, jn = decltype(join_c)::value;
    return p.form_b      ? attend_kernel<1, true, sc, jn>
           : copies == 4 ? attend_kernel<4, false, sc, jn>
           : copies == 2 ? attend_kernel<2, false, sc, jn>
                         : attend_kernel<1, false, sc, jn>;
  };
  using Yes = std::true_type;
  using No = std::false_type;
  auto kernel = score ? (joined ? pick(Yes{}, Yes{}) : pick(Yes{}, No{})) : (joined ? pick(No{}, Yes{}) : pick(No{}, No{}));
  if (!prepare_device(reinterpret_cast<const void*>(kernel), kSmem)) return fail(kStatusCuda, "tree_attn: no usable device");
  cudaError_t e = launch_pdl(kernel, dim3(a.grid), dim3(threads_of(copies)), kSmem, cs,
                             joined ? dim3(a.join, 1, 1) : dim3(0), qm, km, vm, kdm, vdm, a);
  if (e != cudaSuccess) return fail(kStatusCuda, "tree_attn launch: %s", cudaGetErrorString(e));
  const long long blocks = static_cast<long long>(B) * Hkv * p.pairs * (p.form_b ? 2 : 1) * ((p.npt * G + 31) / 32);
  auto join = p.form_b ? (score ? combine_kernel<true, true> : combine_kernel<true, false>)
                       : (score ? combine_kernel<false, true> : combine_kernel<false, false>);
  if (cut) e = launch_pdl(join, dim3(static_cast<unsigned>(blocks), 4), dim3(256), 0, cs, dim3(0), a);
  if (e != cudaSuccess) return fail(kStatusCuda, "tree_attn join launch: %s", cudaGetErrorString(e));
  if (score) {
    ScoreArgs sa{};
    sa.a = a;
    sa.score = node_score;
    sa.tiles = static_cast<int>(tiles);
    // nodes in eights, as many as fit beside the query heads; heads in sixteens beyond that
    sa.gb = G < 16 ? G : 16;
    const int fit = 128 / sa.gb / 8 * 8, all = (T + 7) / 8 * 8;
    sa.chunk = all < fit ? all : fit;
    const int smem = score_smem(T);
    if (!prepare_device(reinterpret_cast<const void*>(score_kernel), score_smem(kMaxNodes)))
      return fail(kStatusCuda, "tree_attn: no usable device");
    // kv heads of a sequence's tile side by side while there are SMs for them
    const int resident = smem <= 76800 ? 3 : smem <= 115712 ? 2 : 1;
    const long long units = tiles * B;
    const long long hs = (static_cast<long long>(resident) * sms + units - 1) / units;
    sa.hsplit = static_cast<int>(hs < 1 ? 1 : hs > Hkv ? Hkv : hs);
    CUtensorMap sqm;
    if ((st = map_rows(&sqm, q, Hq, static_cast<long long>(B) * T, 1, sa.chunk))) return st;
    e = launch_pdl(score_kernel, dim3(static_cast<unsigned>(tiles), sa.hsplit, B), dim3(kScoreThreads), smem, cs,
                   dim3(0), sqm, km, kdm, sa);
    if (e != cudaSuccess) return fail(kStatusCuda, "tree_attn score launch: %s", cudaGetErrorString(e));
  }
  return kStatusOk;
}
