// 8-bit floating point (e4m3) products with one fp32 scale per block of 128,
// on the tcgen05 tensor cores: the dense projection and the routed experts'
// feed-forward, with the quantiser of their activations.
//
// Mathematics.  A row of activations x is cut into blocks of 128 columns; per
// block b, s[b] = max|x| / 448 and q = e4m3(x / s[b]).  A weight matrix W has
// one scale per 128 x 128 block.  A product is
//   y[t][n] = sum_b (s[t][b] * sw[n / 128][b]) * (sum_{k in b} q[t][k] * W[n][k]):
// the inner sums are the tensor cores' (exact products, fp32 sums in tensor
// memory), the outer one fp32 FMAs in registers.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cfloat>
#include <mutex>
#include <set>
#include <utility>

#include "engine.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace lb {

namespace {

constexpr int kF8M = 128;         // weight rows per tile (the MMA's M)
constexpr int kF8Block = 128;     // columns per scale, bytes per staged row
constexpr int kF8EpiWarps = 8;    // two warpgroups, half of the tokens each
constexpr int kF8Threads = (kF8EpiWarps + 3) * 32;
constexpr int kF8Scales = 8;      // ring of staged activation scales
constexpr int kF8MaxBuf = 4;      // ring of accumulators in tensor memory
constexpr int kF8MaxSplit = 8;    // CTAs of a cluster that share a tile's K,
constexpr int kF8SplitBlocks = 3; // with at least this many blocks each
constexpr int kF8StepUnits = 4;   // (row, four blocks) pairs of a warp that quantises, at a time
constexpr int kF8StepEntries = 256;  // entries that a CTA groups for itself
constexpr int kF8StepMost = 48;   // such pairs of a CTA, at most,
constexpr int kF8StepTokens = 32; // and tokens (33 to 64 gained by the smallest matrices alone)

enum F8Mode {
  kF8Out,      // y to out (fp32 or bf16)
  kF8Step,     // the same for few tokens, which every CTA quantises for itself
  kF8Act,      // activation of gate and up, quantised: the down product's input
  kF8StepAct,  // the same for few entries, which every CTA groups and quantises for itself
  kF8Partial,  // y to the row of its (token, rank) entry
  kF8StepPartial,  // the same for few entries, which every CTA groups for itself; the
                   // last CTA of a row block adds up the block's columns of out
};

// e4m3 of v as a byte: round to nearest even, NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3_byte(float v) {
  return (uint32_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

// Four of them, the first in the lowest byte.
__device__ __forceinline__ uint32_t e4m3_word(float2 lo, float2 hi) {
  const uint32_t a = __nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3);
  const uint32_t b = __nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3);
  return __byte_perm(a, b, 0x5410);
}

// max(|a|, |b|, |c|), a NaN if one is.
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}
// The largest of the warp's values, which are not negative; a NaN if one is.
__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// The scale of a block whose largest magnitude has the bits `amax` (a NaN's
// bits are above infinity's, so a maximum over bits keeps a NaN).  A block of
// zeros, or of values too small to scale, takes the smallest normal number.
__device__ __forceinline__ float block_scale(uint32_t amax) {
  const float s = __fdiv_rn(__uint_as_float(amax), 448.0f);
  return s < FLT_MIN ? FLT_MIN : s;
}

// v / s, correctly rounded, with r the correctly rounded 1 / s: with q0 = v * r,
// q0 + r * (v - q0 * s) is it (Markstein, IBM J. Res. Dev. 34, 1990), as long as
// nothing underflows, which holds for the blocks that scale_divides accepts.  A
// quotient a bit off would turn over the ties that bf16 inputs make.
__device__ __forceinline__ float quotient(float v, float s, float r) {
  const float q0 = __fmul_rn(v, r);
  return fmaf(r, fmaf(-q0, s, v), q0);
}
__device__ __forceinline__ bool scale_divides(float s, uint32_t amax) {
  return amax == 0 || (s >= 0x1p-80f && s <= 0x1p100f);
}
// Two values at once.
__device__ __forceinline__ float2 quotient2(float2 v, float2 s_neg, float2 r) {
  const float2 q0 = __fmul2_rn(v, r);
  return __ffma2_rn(r, __ffma2_rn(q0, s_neg, v), q0);
}

// ------------------------------------------------------------ quantiser

// Four consecutive values as they lie in memory, the first n of them where they
// cannot be loaded at once; and as floats.
__device__ __forceinline__ float4 load4(const float* p, bool vec, int n) {
  if (vec) return *reinterpret_cast<const float4*>(p);
  return make_float4(p[0], n > 1 ? p[1] : 0.0f, n > 2 ? p[2] : 0.0f, n > 3 ? p[3] : 0.0f);
}
__device__ __forceinline__ uint2 load4(const __nv_bfloat16* p, bool vec, int n) {
  if (vec) return *reinterpret_cast<const uint2*>(p);
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
  return make_uint2(h[0] | (n > 1 ? (uint32_t)h[1] << 16 : 0u),
                    (n > 2 ? (uint32_t)h[2] : 0u) | (n > 3 ? (uint32_t)h[3] << 16 : 0u));
}
__device__ __forceinline__ void floats4(float4 f, float2 (&v)[2]) {
  v[0] = make_float2(f.x, f.y), v[1] = make_float2(f.z, f.w);
}
__device__ __forceinline__ void floats4(uint2 u, float2 (&v)[2]) {
  v[0] = make_float2(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u));
  v[1] = make_float2(__uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ float4 zero4(const float*) { return make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
__device__ __forceinline__ uint2 zero4(const __nv_bfloat16*) { return make_uint2(0u, 0u); }

// Where a token's quantised row goes: row t, or the grouped rows of its k
// entries (those whose expert is in [0, E)), row_start[expert] + pos[entry].
struct F8Rows {
  const int *sel, *pos, *row_start;  // null: row t
  int* entry;                        // receives the entry of each grouped row
  int k, E;
};

constexpr int kQuantBlocks = 4;  // blocks of one token per warp

// The values of blocks b0 .. b0 + 3 of a row of `cols` columns, zeros past them.
template <typename T, typename Raw>
__device__ __forceinline__ void load_blocks(const T* row, int cols, int b0, bool vec,
                                            Raw (&raw)[kQuantBlocks]) {
  const int c0 = b0 * kF8Block + 4 * (threadIdx.x & 31);
  const T* src = row + c0;
  if (vec && (b0 + kQuantBlocks) * kF8Block <= cols) {
#pragma unroll
    for (int i = 0; i < kQuantBlocks; ++i) raw[i] = load4(src + i * kF8Block, true, 4);
  } else {
#pragma unroll
    for (int i = 0; i < kQuantBlocks; ++i) {
      const int c = c0 + i * kF8Block;
      raw[i] = zero4(row);
      if (c < cols) raw[i] = load4(src + i * kF8Block, vec && c + 4 <= cols, cols - c);
    }
  }
}

// Four blocks of a token, four columns a lane and block: their e4m3 bytes, and
// on lane i the scale of block i (mine: that lane's block exists).
template <typename Raw>
__device__ __forceinline__ void quant_blocks(const Raw (&raw)[kQuantBlocks], bool mine,
                                             uint32_t (&w)[kQuantBlocks], float& s_own) {
  const int lane = threadIdx.x & 31;
  float2 v[kQuantBlocks][2];
  float am = 0.0f;  // lane i: the largest magnitude of block i
#pragma unroll
  for (int i = 0; i < kQuantBlocks; ++i) {
    floats4(raw[i], v[i]);
    const float m = warp_max_nan(
        max_abs3(max_abs3(v[i][0].x, v[i][0].y, v[i][1].x), v[i][1].y, 0.0f));
    if (lane == i) am = m;
  }
  // am / 448 as a quotient by the rounded reciprocal; where that or the
  // values' own do not hold, the slow way
  s_own = quotient(am, 448.0f, 1.0f / 448.0f);
  const bool plain =
      __all_sync(0xffffffffu, !mine || am == 0.0f || (am >= 0x1p-70f && am <= 0x1p100f));
  if (am == 0.0f) s_own = FLT_MIN;
  if (!plain) s_own = block_scale(__float_as_uint(am));
  if (plain) {
    const float r_own = __frcp_rn(s_own);
#pragma unroll
    for (int i = 0; i < kQuantBlocks; ++i) {
      const float s = __shfl_sync(0xffffffffu, s_own, i), r = __shfl_sync(0xffffffffu, r_own, i);
      const float2 s2 = make_float2(-s, -s), r2 = make_float2(r, r);
      w[i] = e4m3_word(quotient2(v[i][0], s2, r2), quotient2(v[i][1], s2, r2));
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < kQuantBlocks; ++i) {
      const float s = __shfl_sync(0xffffffffu, s_own, i);
      uint32_t wi = 0;
#pragma unroll
      for (int ii = 0; ii < kQuantBlocks; ++ii)
        if (ii == i)
          wi = e4m3_word(make_float2(__fdiv_rn(v[ii][0].x, s), __fdiv_rn(v[ii][0].y, s)),
                         make_float2(__fdiv_rn(v[ii][1].x, s), __fdiv_rn(v[ii][1].y, s)));
#pragma unroll
      for (int ii = 0; ii < kQuantBlocks; ++ii)
        if (ii == i) w[ii] = wi;
    }
  }
}

// One warp per token and kQuantBlocks blocks of 128 columns, four columns a
// lane and block, every load issued before the first is used.  q has rows of
// q_pitch bytes (a multiple of 16, zeros past cols), scales the layout
// [block][s_pitch] the products read with bulk copies; ungrouped, the scales
// of rows [tokens, s_pitch) are zeroed.
//
// Bound by memory, and nearly by issue: the four blocks' scales are computed
// side by side on the lanes, one reciprocal for all, and values are divided two
// at a time.  8192 x 4096 bf16: 47 us with a division a value, 25 with
// quotients by the reciprocal one at a time, 21 now; warps that stay and
// request the next token's values ahead took 27.
template <typename T, bool GROUPED>
__global__ void __launch_bounds__(256) f8_quant_kernel(const T* __restrict__ x, long ldx,
                                                       int tokens, int cols, uint8_t* q,
                                                       int q_pitch, float* scales, int s_pitch,
                                                       F8Rows rows, int vec) {
  using Raw = decltype(load4(x, true, 4));
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31;
  const int blocks = (cols + kF8Block - 1) / kF8Block;
  const unsigned per = (blocks + kQuantBlocks - 1) / kQuantBlocks;
  const unsigned unit = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = (int)(unit / per), b0 = (int)(unit - t * per) * kQuantBlocks;
  const int c0 = b0 * kF8Block + 4 * lane;
  const bool whole = (b0 + kQuantBlocks) * kF8Block <= cols;
  const bool mine = lane < kQuantBlocks && b0 + lane < blocks;  // this lane's scale exists
  uint8_t* dst = q + c0;
  float* sp = scales + (long)(b0 + lane) * s_pitch;
  if (t >= tokens) {
    if (!GROUPED && t < s_pitch && mine) sp[t] = 0.0f;
    return;
  }
  Raw raw[kQuantBlocks];
  load_blocks(x + t * ldx, cols, b0, vec, raw);
  uint32_t w[kQuantBlocks];
  float s_own;
  quant_blocks(raw, mine, w, s_own);
  auto store = [&](uint8_t* row, float* scale) {
    uint32_t* out = reinterpret_cast<uint32_t*>(row);
    if (whole) {
#pragma unroll
      for (int i = 0; i < kQuantBlocks; ++i) out[i * (kF8Block / 4)] = w[i];
    } else {
#pragma unroll
      for (int i = 0; i < kQuantBlocks; ++i)
        if (c0 + i * kF8Block < q_pitch) out[i * (kF8Block / 4)] = w[i];
    }
    if (mine) *scale = s_own;
  };
  if (!GROUPED) {
    store(dst + (long)t * q_pitch, sp + t);
  } else {
    for (int j0 = 0; j0 < rows.k; j0 += 32) {  // the entries' rows, one a lane
      const int id = t * rows.k + j0 + lane;
      int o = -1;
      if (j0 + lane < rows.k) {
        const int e = __ldg(rows.sel + id);
        if (e >= 0 && e < rows.E) o = __ldcg(rows.row_start + e) + __ldcg(rows.pos + id);
      }
      if (b0 == 0 && o >= 0) rows.entry[o] = id;
      for (int j = 0; j < min(32, rows.k - j0); ++j) {
        const int oj = __shfl_sync(0xffffffffu, o, j);
        if (oj >= 0) store(dst + (long)oj * q_pitch, sp + oj);
      }
    }
  }
}

// ------------------------------------------------------------ products

struct F8Maps {
  CUtensorMap x, w0, w1;
};

struct F8Pass {
  int rows, rblocks, kblocks;    // weight rows of one expert, their blocks, blocks of K
  const float *ws0, *ws1;        // weight scales [expert][rblocks][kblocks]
  const float* xs;               // activation scales [kblocks][xs_pitch]
  long xs_pitch;
  int tokens, chunks;            // dense: rows of x and their tiles of NT
  const int4* tiles;             // grouped: {first row, rows, expert, 0} of each chunk,
  const int* nchunks;            //   null when dense
  const void* x;                 // kF8Step, kF8StepAct: the rows themselves
  long ldx;
  int cols, x_bf16, x_vec;
  // few entries: their number, and a counter for each row block of the down
  // product (kF8StepAct zeroes the nclear counters)
  int n, nclear;
  int* counters;
  void* out;                     // kF8Out, kF8Step, kF8StepPartial
  long ldo;
  int out_bf16;
  uint8_t* hq;                   // kF8Act: quantised activations and their scales
  long h_pitch;
  float* hs;
  long hs_pitch;
  float* partial;                // kF8Partial: rows of partial by entry
  long ldp;
  const int* entry;
  const int* sel;
  const float* weights;
  int k, E;
  int pairs;                     // CTA pairs of the device (large products)
  int split;                     // CTAs of a cluster share a tile's K (1: no cluster)
  int early;                     // the weights and tiles are not the previous kernel's output
  int* status;
};

struct F8Sync {
  uint64_t full[16], empty[16];
  uint64_t sfull[kF8Scales], sempty[kF8Scales];
  uint64_t tfull[kF8MaxBuf], tempty[kF8MaxBuf], done, xfull;
  uint32_t tmem;
  int abort, last;
};

// kF8StepAct, kF8StepPartial: the grouping of up to kF8StepEntries entries by
// expert, as f8_plan_kernel has it, and this CTA's tile of it.
struct F8Group {
  int e[kF8StepEntries], count[kF8StepEntries], row[kF8StepEntries];
  int ent[16], tok[16];  // entry and token of each row of the tile
  int chunks, row0, rows, expert;
};

// Small tiles are bound by the weights' bytes: two CTAs a multiprocessor, so
// that one loads while the other finishes a tile.  Large ones take the whole
// shared memory for one, as does kF8Step with every block of its tokens.
template <int NT, int MATS, int MODE>
struct F8Cfg {
  static constexpr bool kStep = MODE == kF8Step || MODE == kF8StepAct;
  static constexpr bool kGroup = MODE == kF8StepAct || MODE == kF8StepPartial;
  static constexpr bool kPartial = MODE == kF8Partial || MODE == kF8StepPartial;
  static constexpr int kCtas = MODE == kF8Step || (NT == 64 && MATS == 2) ? 1 : 2;
  static constexpr uint32_t kA = kF8M * kF8Block;        // bytes of one weight tile
  static constexpr uint32_t kX = NT * kF8Block;          // and of one block of activations
  static constexpr uint32_t kStage = MATS * kA + (kStep ? 0 : kX);
  static constexpr uint32_t kBudget =
      MODE == kF8Step ? 5 * kStage : kStep ? 64u * 1024u : (kCtas == 2 ? 104u : 200u) * 1024u;
  static constexpr int kStages = (int)(kBudget / kStage);
  // blocks of K a CTA quantises, at most: kF8StepAct leaves room for a CTA of the
  // down product, which requests its weights while it waits
  static constexpr int kStepBlocks = MODE == kF8Step ? 128 * 1024 / (int)kX : 21;
  static constexpr uint32_t kAcc = NT * MATS;            // tensor-memory columns of one buffer
  static constexpr int kBufs = 512 / kAcc / kCtas > kF8MaxBuf ? kF8MaxBuf : 512 / kAcc / kCtas;
  static constexpr uint32_t kCols = kBufs * kAcc < 32 ? 32 : kBufs * kAcc;
  static constexpr int kScales = kStep ? kStepBlocks : kF8Scales;  // blocks of scales staged
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + (kStep ? kStepBlocks * kX : 0) +
                                  kScales * NT * 4 + 2 * 4 * NT * 4 + sizeof(F8Sync) +
                                  (kGroup ? sizeof(F8Group) : 0);
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

// Instruction descriptor, kind::f8f6f4: fp32 accumulator (bits 4-5 = 1), A and
// B e4m3 (bits 7-9 and 10-12 = 0), both K-major, N >> 3 in bits 17-22, M >> 4
// in bits 24-28.
__device__ __forceinline__ uint32_t f8_idesc(int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kF8M >> 4) << 24);
}

// D[tmem] (+)= A[smem] . B[smem]^T over 32 columns of K.
__device__ __forceinline__ void tc_mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                          uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(void* dst, const void* tmap, int x, int y, int z,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3, %4}], [%5];" ::"r"(smem_addr(dst)),
      "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}

// 8 consecutive fp32 columns of this thread's tensor-memory lane (no wait).
__device__ __forceinline__ void tmem_ld8_issue(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
// Waits for this thread's tensor-memory loads; the registers pass through so
// that no use of them moves above the wait.
__device__ __forceinline__ void tmem_wait_ld8(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}

// Bounded wait of the product kernel's pipelines: a try_wait without a time
// hint returns as soon as the phase completes.
__device__ __forceinline__ bool f8_wait(uint64_t* bar, uint32_t parity, int* status,
                                        volatile int* abort) {
  auto attempt = [&] {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n "
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    return ok != 0;
  };
  if (attempt()) return true;
  const uint64_t t0 = global_ns();
  for (;;) {
    for (int i = 0; i < 16; ++i)
      if (attempt()) return true;
    if (*abort) return false;
    if (global_ns() - t0 >= kWaitLimitNs) break;
  }
  if (status) atomicOr(status, 2);
  *abort = 1;
  return false;
}

// After a wait that gave up: copies that are still in flight land before the
// CTA's memory goes (otherwise the MMAs have waited for every copy).
__device__ __forceinline__ void f8_linger() {
  const uint64_t t0 = global_ns();
  while (global_ns() - t0 < 1000000) {
  }
}

// f8_wait by a whole warp, with a result that is the same on every lane.
__device__ __forceinline__ bool f8_wait_warp(uint64_t* bar, uint32_t parity, int* status,
                                             volatile int* abort) {
  return __all_sync(0xffffffffu, f8_wait(bar, parity, status, abort));
}

__device__ __forceinline__ void store_out(void* out, int bf16, long i, float v) {
  if (bf16)
    static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
  else
    static_cast<float*>(out)[i] = v;
}

// One column of token t's weighted sum over its entries, in rank order; entries
// whose expert is outside [0, E) add nothing.  partial: that column of entry 0.
__device__ __forceinline__ float combine_column(const float* partial, long ldp, const int* sel,
                                                int E, const float* weights, int t, int k) {
  float a = 0.0f;
#pragma unroll 8
  for (int j = 0; j < k; ++j) {
    const int e = sel[t * k + j];
    if (e >= 0 && e < E)
      a = fmaf(weights[t * k + j], __ldcg(partial + (long)(t * k + j) * ldp), a);
  }
  return a;
}

struct F8Tile {
  int row0, count, expert, rb;  // first row of x, valid rows, expert, row block
};

// Tiles in the order the CTAs take them.  Dense: the token chunks of one row
// block next to each other, so its weights come from L2 after the first.
// Grouped: the row blocks of one chunk next to each other.
template <int NT>
__device__ __forceinline__ F8Tile f8_tile(const F8Pass& p, int tile) {
  F8Tile t;
  if (p.tiles) {
    const int c = tile / p.rblocks;
    const int4 v = __ldcg(p.tiles + c);
    t.row0 = v.x, t.count = v.y, t.expert = v.z, t.rb = tile - c * p.rblocks;
  } else {
    t.rb = tile / p.chunks;
    t.row0 = (tile - t.rb * p.chunks) * NT;
    t.count = min(NT, p.tokens - t.row0);
    t.expert = 0;
  }
  return t;
}

// (__fdividef is off by two steps at most; for a divisor above 2^126 it gives 0,
// where the exact quotient is below 2^-119)
__device__ __forceinline__ float silu(float g) { return __fdividef(g, 1.0f + expf(-g)); }

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
// The cluster address of the same shared-memory object in its CTA `rank`.
__device__ __forceinline__ uint32_t cluster_map(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float cluster_ld(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Groups the entries (token t, rank j; id t * k + j) by expert, in every CTA for
// itself, as f8_plan_kernel does: entry i counts the entries of its expert
// before it and in all, then the rows and chunks (of NT) of the experts before
// its own.  Entries whose expert is outside [0, E) are in no group.  Leaves the
// rows of chunk `mine`, their entries and tokens in g (rows 0: there is no such
// chunk).
template <int NT>
__device__ __forceinline__ void step_group(const F8Pass& p, F8Group& g, int mine) {
  const int i = threadIdx.x;
  const bool on = i < kF8StepEntries;
  int e = on && i < p.n ? __ldcg(p.sel + i) : -1;
  if (e >= p.E) e = -1;
  if (on) g.e[i] = e;
  if (i == 0) g.chunks = g.row0 = g.rows = g.expert = 0;
  __syncthreads();
  int pos = 0, cnt = 0;
  if (on)
    for (int j = 0; j < p.n; ++j) {
      const bool same = g.e[j] == e;
      pos += same && j < i;
      cnt += same;
    }
  const bool first = e >= 0 && pos == 0;
  if (on) g.count[i] = first ? cnt : 0;
  __syncthreads();
  int base = 0, chunk = 0;
  if (on) {
    for (int j = 0; j < p.n; ++j) {
      const int c = g.e[j] < e ? g.count[j] : 0;
      base += (c + 3) & ~3;
      chunk += (c + NT - 1) / NT;
    }
    g.row[i] = e >= 0 ? base + pos : -1;
  }
  const int ch = (cnt + NT - 1) / NT;
  if (first) {
    atomicMax(&g.chunks, chunk + ch);
    const int c = mine - chunk;
    if (c >= 0 && c < ch) g.row0 = base + c * NT, g.rows = min(NT, cnt - c * NT), g.expert = e;
  }
  __syncthreads();
  if (on && g.row[i] >= g.row0 && g.row[i] < g.row0 + g.rows) {
    g.ent[g.row[i] - g.row0] = i;
    g.tok[g.row[i] - g.row0] = i / p.k;
  }
  __syncthreads();
}

// kF8Step, kF8StepAct: blocks [kb0, kb1) of `rows` rows (row r is token tok[r],
// or r without tok), by the eight epilogue warps, into shared memory as a TMA
// copy with the 128-byte swizzle would lay them out (16 bytes' place within a
// row of 128 exclusive-or the row's number modulo 8).  Rows past the last keep
// what they hold: they reach no column that is stored.
template <int NT, int UNITS, typename T>
__device__ __forceinline__ void step_quantize(const F8Pass& p, const T* x, int rows, const int* tok,
                                              int kb0, int kb1, uint8_t* s_x, float* s_scale) {
  using Raw = decltype(load4(x, true, 4));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (kb1 - kb0 + kQuantBlocks - 1) / kQuantBlocks, units = rows * per;
  for (int u0 = warp; u0 < units; u0 += UNITS * kF8EpiWarps) {
    Raw raw[UNITS][kQuantBlocks];
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {  // these units' loads before the first is used
      const int u = u0 + i * kF8EpiWarps, r = u / per;
      if (u < units)
        load_blocks(x + (long)(tok ? tok[r] : r) * p.ldx, p.cols, kb0 + (u - r * per) * kQuantBlocks,
                    p.x_vec, raw[i]);
    }
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int u = u0 + i * kF8EpiWarps, r = u / per, b0 = (u - r * per) * kQuantBlocks;
      if (u >= units) break;
      const bool mine = lane < kQuantBlocks && kb0 + b0 + lane < kb1;
      uint32_t w[kQuantBlocks];
      float s;
      quant_blocks(raw[i], mine, w, s);
#pragma unroll
      for (int j = 0; j < kQuantBlocks; ++j)
        if (kb0 + b0 + j < kb1)
          *reinterpret_cast<uint32_t*>(s_x + (b0 + j) * (NT * kF8Block) + r * kF8Block +
                                       (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) = w[j];
      if (mine) s_scale[(b0 + lane) * NT + r] = s;
    }
  }
}

// Persistent over tiles of 128 weight rows x NT rows of x (M is the weights'
// side, so one token costs a tile of 16 columns, and an expert's few tokens no
// more).  Warp 8 stages weights and activations by TMA, warp 10 the activations'
// scales, warp 9's first lane issues the MMAs of one block of K into the next
// of kBufs accumulators, and warps 0-7 add the accumulators, scaled, into
// registers: lane r of the tensor memory is weight row r, so the weight scale
// is one number per block and thread.
//
// SPLIT: few tiles.  The CTAs of a cluster take a part of the tile's K
// each, then each adds the sums of its share of the columns from the others'
// shared memory.
template <int NT, int MATS, int MODE, bool SPLIT>
__global__ void __launch_bounds__(kF8Threads, (F8Cfg<NT, MATS, MODE>::kCtas))
    f8_gemm_kernel(const __grid_constant__ F8Maps maps, const F8Pass p) {
  using C = F8Cfg<NT, MATS, MODE>;
  constexpr int NC = NT / 2;  // tokens per epilogue thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint8_t* s_x = stages + (size_t)C::kStages * C::kStage;  // kF8Step: [block][NT][128], swizzled
  float* s_scale = reinterpret_cast<float*>(s_x + (C::kStep ? C::kStepBlocks * C::kX : 0));
  uint32_t* s_amax = reinterpret_cast<uint32_t*>(s_scale + C::kScales * NT);  // [parity][quadrant][NT]
  F8Sync* sy = reinterpret_cast<F8Sync*>(s_amax + 2 * 4 * NT);
  F8Group* sg = reinterpret_cast<F8Group*>(sy + 1);
  volatile int* abort = &sy->abort;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&sy->full[s], 1);
      mbar_init(&sy->empty[s], 1);
    }
    for (int s = 0; s < kF8Scales; ++s) {
      mbar_init(&sy->sfull[s], 1);
      mbar_init(&sy->sempty[s], kF8EpiWarps);
    }
    for (int b = 0; b < C::kBufs; ++b) {
      mbar_init(&sy->tfull[b], 1);
      mbar_init(&sy->tempty[b], kF8EpiWarps);
    }
    mbar_init(&sy->done, 1);
    mbar_init(&sy->xfull, kF8EpiWarps);
    sy->abort = 0;
    fence_mbar_init();
  }
  if (warp == kF8EpiWarps + 1) tmem_alloc(&sy->tmem, C::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sy->tmem, 0);
  const uint32_t rank = SPLIT ? cluster_rank() : 0;
  const int split = SPLIT ? p.split : 1;
  const int tile0 = (int)blockIdx.x / split, tstep = (int)gridDim.x / split;
  // the entries are not the kernel before's output when that is kF8StepAct, which has read them
  if constexpr (MODE == kF8StepPartial) step_group<NT>(p, *sg, tile0 / p.rblocks);
  const bool early = p.early && warp == kF8EpiWarps;
  if (!early) {
    griddep_wait();
    griddep_launch();
  }
  if constexpr (MODE == kF8StepAct) {
    step_group<NT>(p, *sg, tile0 / p.rblocks);
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i < p.nclear; i += kF8Threads) p.counters[i] = 0;
  }
  const int ntiles =
      (C::kGroup ? sg->chunks : p.tiles ? __ldcg(p.nchunks) : p.chunks) * p.rblocks;
  // (kGroup: one tile a CTA at most)
  auto tile_at = [&](int tile) {
    return C::kGroup ? F8Tile{sg->row0, sg->rows, sg->expert, tile % p.rblocks}
                     : f8_tile<NT>(p, tile);
  };
  const int kb0 = (int)rank * p.kblocks / split, kb1 = ((int)rank + 1) * p.kblocks / split;
  bool synced = false;  // split: this warp has met the others of the cluster

  if (warp == kF8EpiWarps) {  // ------------------------------------- weights, activations
    const bool one = elect_one();
    RingPos rp;
    int q = 0, ahead = 0;
    auto load_weights = [&](int s, int kb, const F8Tile& t) {
      uint8_t* st = stages + (size_t)s * C::kStage;
      uint64_t* bar = &sy->full[s];
      mbar_expect_tx(bar, C::kStage);
      tma_load_3d(st, &maps.w0, kb * kF8Block, t.rb * kF8M, t.expert, bar);
      if (MATS == 2)
        tma_load_3d(st + C::kA, &maps.w1, kb * kF8Block, t.rb * kF8M, t.expert, bar);
    };
    if (early) {  // the first tile's weights while the previous kernel still runs
      if (tile0 < ntiles) {
        const F8Tile t = tile_at(tile0);
        for (; ahead < C::kStages && kb0 + ahead < kb1; ++ahead)
          if (one) load_weights(ahead, kb0 + ahead, t);
      }
      griddep_wait();
      griddep_launch();
    }
    bool ok = true;
    for (int tile = tile0; tile < ntiles && ok; tile += tstep) {
      const F8Tile t = tile_at(tile);
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = q < C::kStages || f8_wait_warp(&sy->empty[rp.s], rp.phase ^ 1u, p.status, abort);
        if (!ok) break;
        if (one) {
          if (q >= ahead) load_weights(rp.s, kb, t);
          if (!C::kStep)
            tma_load_2d(stages + (size_t)rp.s * C::kStage + MATS * C::kA, &maps.x, kb * kF8Block,
                        t.row0, &sy->full[rp.s]);
        }
        ++q;
        rp.next(C::kStages);
      }
    }
    __syncwarp();
  } else if (warp == kF8EpiWarps + 2) {  // -------------------------------------------- scales
    const bool one = elect_one();
    RingPos rp;
    int q = 0;
    bool ok = !C::kStep;
    for (int tile = tile0; tile < ntiles && ok; tile += tstep) {
      const F8Tile t = tile_at(tile);
      // row0 and the pitch are multiples of 4; columns past the pitch keep
      // what an earlier tile left and belong to no valid row
      const uint32_t bytes = (uint32_t)min((long)NT, p.xs_pitch - t.row0) * 4u;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = q < kF8Scales || f8_wait_warp(&sy->sempty[rp.s], rp.phase ^ 1u, p.status, abort);
        if (!ok) break;
        if (one) {
          mbar_expect_tx(&sy->sfull[rp.s], bytes);
          tma_load_1d(s_scale + rp.s * NT, p.xs + kb * p.xs_pitch + t.row0, bytes,
                      &sy->sfull[rp.s]);
        }
        ++q;
        rp.next(kF8Scales);
      }
    }
    __syncwarp();
  } else if (warp == kF8EpiWarps + 1) {  // ----------------------------------------------- MMA
    const bool one = elect_one();
    RingPos rp, ap;
    int q = 0;
    bool ok = true;
    const uint64_t desc = sw128_desc(stages), xdesc = sw128_desc(s_x);
    if (C::kStep) ok = f8_wait_warp(&sy->xfull, 0, p.status, abort);
    for (int tile = tile0; tile < ntiles && ok; tile += tstep) {
      const F8Tile t = tile_at(tile);
      const uint32_t idesc = f8_idesc((t.count + 15) & ~15);
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = (q < C::kBufs || f8_wait_warp(&sy->tempty[ap.s], ap.phase ^ 1u, p.status, abort)) &&
             f8_wait_warp(&sy->full[rp.s], rp.phase, p.status, abort);
        if (!ok) break;
        tc_fence_after();
        const uint64_t ad = desc + (uint32_t)rp.s * (C::kStage >> 4);
        const uint64_t bd = C::kStep ? xdesc + (uint32_t)(kb - kb0) * (C::kX >> 4)
                                     : ad + (MATS * C::kA >> 4);
        const uint32_t d = tmem + ap.s * C::kAcc;
        if (one) {
#pragma unroll
          for (int mat = 0; mat < MATS; ++mat)
#pragma unroll
            for (int j = 0; j < 4; ++j)  // K steps of 32 bytes
              tc_mma_f8(d + mat * NT, ad + mat * (C::kA >> 4) + 2 * j, bd + 2 * j, idesc, j != 0);
          tc_commit(&sy->empty[rp.s]);
          tc_commit(&sy->tfull[ap.s]);
        }
        __syncwarp();
        ++q;
        rp.next(C::kStages);
        ap.next(C::kBufs);
      }
    }
    // every MMA issued has completed before the tensor memory is freed
    if (one) tc_commit(&sy->done);
    mbar_wait(&sy->done, 0, nullptr);
    __syncwarp();
  } else {  // ------------------------------------------ epilogue
    const int quad = warp & 3, half = warp >> 2, r = 32 * quad + lane;
    const uint32_t lane_base = (uint32_t)(32 * quad) << 16;
    RingPos ap, sp;
    bool ok = true;
    int parity = 0;
    if constexpr (C::kStep) {
      // (an expert of few entries has a row or two: one unit a warp mostly)
      constexpr int kUnits = MODE == kF8StepAct ? 1 : kF8StepUnits;
      const int rows = MODE == kF8StepAct ? sg->rows : p.tokens;
      const int* tok = MODE == kF8StepAct ? sg->tok : nullptr;
      if (p.x_bf16)
        step_quantize<NT, kUnits>(p, static_cast<const __nv_bfloat16*>(p.x), rows, tok, kb0, kb1,
                                  s_x, s_scale);
      else
        step_quantize<NT, kUnits>(p, static_cast<const float*>(p.x), rows, tok, kb0, kb1, s_x,
                                  s_scale);
      fence_proxy_async_smem();  // the MMAs read what these threads wrote
      __syncwarp();
      if (lane == 0) mbar_arrive(&sy->xfull);
      named_bar_sync(3, kF8EpiWarps * 32);  // and all of them the scales
    }
    if (MODE == kF8StepPartial && ntiles == 0)  // no entry is anyone's
      for (long i = (long)blockIdx.x * kF8EpiWarps * 32 + threadIdx.x; i < (long)p.tokens * p.rows;
           i += (long)gridDim.x * kF8EpiWarps * 32)
        store_out(p.out, p.out_bf16, i / p.rows * p.ldo + i % p.rows, 0.0f);
    for (int tile = tile0; tile < ntiles && ok; tile += tstep, parity ^= 1) {
      const F8Tile t = tile_at(tile);
      // this thread's tokens: groups of 8 columns in turn with the other half's,
      // so that both have their share of a tile that is not full
      auto col = [&](int c) { return (2 * (c >> 3) + half) * 8 + (c & 7); };
      auto in = [&](int c) { return col(c) < t.count; };
      const long ws_row = ((long)t.expert * p.rblocks + t.rb) * p.kblocks;
      float2 acc[MATS][NC / 2];
#pragma unroll
      for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int c = 0; c < NC / 2; ++c) acc[m][c] = make_float2(0.0f, 0.0f);
      auto own = [&](int c) { return !SPLIT || (c & (p.split - 1)) == (int)rank; };
      float wl[MATS];  // weight scales of 32 blocks, one a lane
      int ent[(NC + 31) / 32];  // entries of this thread's tokens, 32 a register
      if (C::kPartial) {
#pragma unroll
        for (int i = 0; i < (NC + 31) / 32; ++i)
          ent[i] = 32 * i + lane >= NC || !in(32 * i + lane) ? 0
                   : MODE == kF8StepPartial ? sg->ent[col(32 * i + lane)]
                                            : __ldcg(p.entry + t.row0 + col(32 * i + lane));
      }
      for (int kb = kb0; kb < kb1; ++kb) {
        if (((kb - kb0) & 31) == 0) {
          const bool more = kb + lane < kb1;
          wl[0] = more ? __ldg(p.ws0 + ws_row + kb + lane) : 0.0f;
          if (MATS == 2) wl[MATS - 1] = more ? __ldg(p.ws1 + ws_row + kb + lane) : 0.0f;
        }
        float sw[MATS];
#pragma unroll
        for (int m = 0; m < MATS; ++m) sw[m] = __shfl_sync(0xffffffffu, wl[m], (kb - kb0) & 31);
        ok = (C::kStep || f8_wait(&sy->sfull[sp.s], sp.phase, p.status, abort)) &&
             f8_wait(&sy->tfull[ap.s], ap.phase, p.status, abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const float* sc = s_scale + (C::kStep ? kb - kb0 : sp.s) * NT;
        // columns loaded together, as many as the registers hold: the loads of a
        // second group wait for the first
        constexpr int CH = C::kCtas == 2 ? (NC < 16 / MATS ? NC : 16 / MATS)
                                         : (NC < 64 / MATS ? NC : 64 / MATS);
#pragma unroll
        for (int c0 = 0; c0 < NC; c0 += CH) {
          if (in(c0)) {  // warp-uniform
            uint32_t d[MATS][CH];
#pragma unroll
            for (int m = 0; m < MATS; ++m)
#pragma unroll
              for (int j = 0; j < CH; j += 8)
                tmem_ld8_issue(tmem + lane_base + ap.s * C::kAcc + m * NT + col(c0 + j), d[m] + j);
#pragma unroll
            for (int m = 0; m < MATS; ++m)
#pragma unroll
              for (int j = 0; j < CH; j += 8) tmem_wait_ld8(d[m] + j);
#pragma unroll
            for (int j = 0; j < CH; j += 4) {
              const float4 sx = *reinterpret_cast<const float4*>(sc + col(c0 + j));
#pragma unroll
              for (int m = 0; m < MATS; ++m) {
                const float2 w = make_float2(sw[m], sw[m]);
                acc[m][(c0 + j) / 2] =
                    __ffma2_rn(make_float2(__uint_as_float(d[m][j]), __uint_as_float(d[m][j + 1])),
                               __fmul2_rn(make_float2(sx.x, sx.y), w), acc[m][(c0 + j) / 2]);
                acc[m][(c0 + j) / 2 + 1] = __ffma2_rn(
                    make_float2(__uint_as_float(d[m][j + 2]), __uint_as_float(d[m][j + 3])),
                    __fmul2_rn(make_float2(sx.z, sx.w), w), acc[m][(c0 + j) / 2 + 1]);
              }
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sy->tempty[ap.s]);
          if (!C::kStep) mbar_arrive(&sy->sempty[sp.s]);
        }
        ap.next(C::kBufs);
        sp.next(kF8Scales);
      }
      if (!ok) break;
      if (SPLIT) {
        // every product of this CTA is in registers, so the stages are free; CTA
        // `rank` finishes the columns that are `rank` modulo split, adding the
        // CTAs' sums in rank order whoever adds them
        float* red = reinterpret_cast<float*>(stages) + r;
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
          for (int c = 0; c < NC; ++c)
            if (in(c) && !own(c))
              red[(m * NT + col(c)) * kF8M] = c & 1 ? acc[m][c / 2].y : acc[m][c / 2].x;
        cluster_sync();
        synced = true;
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
          for (int c = 0; c < NC; ++c)
            if (in(c) && own(c)) {  // warp-uniform
              const float here = c & 1 ? acc[m][c / 2].y : acc[m][c / 2].x;
              float v[kF8MaxSplit];
#pragma unroll
              for (int k = 0; k < kF8MaxSplit; ++k)
                if (k < split && k != (int)rank)
                  v[k] = cluster_ld(cluster_map(red + (m * NT + col(c)) * kF8M, k));
              float y = 0.0f;
#pragma unroll
              for (int k = 0; k < kF8MaxSplit; ++k)
                if (k < split) y += k == (int)rank ? here : v[k];
              if (c & 1)
                acc[m][c / 2].y = y;
              else
                acc[m][c / 2].x = y;
            }
      }
      const int row = t.rb * kF8M + r;
      if (MODE == kF8Out || MODE == kF8Step) {
        if (row < p.rows) {
#pragma unroll
          for (int c = 0; c < NC; ++c)
            if (in(c) && own(c)) {
              const float y = c & 1 ? acc[0][c / 2].y : acc[0][c / 2].x;
              store_out(p.out, p.out_bf16, (long)(t.row0 + col(c)) * p.ldo + row, y);
            }
        }
      } else if (C::kPartial) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (in(c) && own(c)) {  // warp-uniform
            const float y = c & 1 ? acc[0][c / 2].y : acc[0][c / 2].x;
            const long id = __shfl_sync(0xffffffffu, ent[c / 32], c & 31);
            if (row < p.rows) p.partial[id * p.ldp + row] = y;
          }
        if (MODE == kF8StepPartial) {
          __threadfence();
          named_bar_sync(3, kF8EpiWarps * 32);
          if (threadIdx.x == 0)
            sy->last = atomicAdd(p.counters + t.rb, 1) == ntiles / p.rblocks * split - 1;
          named_bar_sync(3, kF8EpiWarps * 32);
          if (sy->last) {
            __threadfence();
            const int c = t.rb * kF8M + (threadIdx.x & (kF8M - 1));
            if (c < p.rows)
              for (int tok = threadIdx.x / kF8M; tok < p.tokens; tok += kF8EpiWarps * 32 / kF8M)
                store_out(p.out, p.out_bf16, tok * p.ldo + c,
                          combine_column(p.partial + c, p.ldp, p.sel, p.E, p.weights, tok, p.k));
          }
        }
      } else {
        // the 128 rows of this tile are one block of the next product's K: its
        // scale per token is a maximum over the four warps of this half, and
        // lane c works out the scale and its reciprocal of column c (and c + 32)
        uint32_t* am = s_amax + parity * 4 * NT;
        float h[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (in(c) && own(c)) {
            const float u = c & 1 ? acc[MATS - 1][c / 2].y : acc[MATS - 1][c / 2].x;
            const float g = c & 1 ? acc[0][c / 2].y : acc[0][c / 2].x;
            if (MATS == 2) {
              h[c] = silu(g) * u;
            } else {
              const float v = u < 0.0f ? 0.0f : u;  // a NaN stays
              h[c] = v * v;
            }
            if (row >= p.rows) h[c] = 0.0f;
            const uint32_t a =
                __reduce_max_sync(0xffffffffu, __float_as_uint(h[c]) & 0x7fffffffu);
            if (lane == 0) am[quad * NT + col(c)] = a;
          }
        named_bar_sync(1 + half, 128);
        float hs[(NC + 31) / 32], hr[(NC + 31) / 32];
        bool plain = true;
#pragma unroll
        for (int i = 0; i < (NC + 31) / 32; ++i) {
          const int c = 32 * i + lane;
          hs[i] = hr[i] = 0.0f;
          if (c < NC && in(c) && own(c)) {
            const uint32_t* a = am + col(c);
            const uint32_t top = max(max(a[0], a[NT]), max(a[2 * NT], a[3 * NT]));
            hs[i] = block_scale(top);
            hr[i] = __frcp_rn(hs[i]);
            plain = plain && scale_divides(hs[i], top);
            if (quad == 0) p.hs[t.rb * p.hs_pitch + t.row0 + col(c)] = hs[i];
          }
        }
        plain = __all_sync(0xffffffffu, plain);
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (in(c) && own(c)) {
            const float sc = __shfl_sync(0xffffffffu, hs[c / 32], c & 31);
            const float rc = __shfl_sync(0xffffffffu, hr[c / 32], c & 31);
            const float v = plain ? quotient(h[c], sc, rc) : __fdiv_rn(h[c], sc);
            p.hq[(long)(t.row0 + col(c)) * p.h_pitch + row] = (uint8_t)e4m3_byte(v);
          }
      }
    }
  }
  if (*abort) f8_linger();
  if (SPLIT) {
    __syncwarp();
    if (!synced) cluster_sync();
    cluster_sync();  // the others have read this CTA's sums
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kF8EpiWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kCols);
  }
}

// ------------------------------------------------------------ large products

// Many tokens: tiles of 256 tokens x 256 weight rows, each by a pair of CTAs
// (cta_group::2).  CTA r of the pair stages tokens [128 r, 128 r + 128) and
// weight rows [128 r, 128 r + 128) of the tile, 32 KB a block of K; the pair's
// MMA reads both and leaves 128 tokens x 256 columns of fp32 sums in each CTA's
// tensor memory, twice, so that a block's MMAs run while the one before is
// added up.  What bounds small tiles of many tokens is the way from L2: one of
// 128 x 64 reads 24 KB a block for an eighth of a pair's products (2048 tokens by
// 14336 x 8192: 453 us in small tiles, 244 in pairs).
//
// Here M is the tokens' side: a thread of the epilogue has one token and 64
// columns of one weight block, so a block of K has one factor a thread and 32
// packed FMAs are about all it costs.
constexpr int kBigStages = 4;
constexpr int kBigEpi = 16;  // epilogue warps: a tile's 256 columns in four parts
constexpr int kBigThreads = (kBigEpi + 2) * 32;
constexpr uint32_t kBigStage = 2 * kF8M * kF8Block;
constexpr int kBigPitch = 17;  // words of a row staged for plain stores, one more than it holds
constexpr int kBigRow = 128;   // bytes of one staged for a bulk copy,
constexpr int kBigRowPitch = kBigRow + 16;  // and between two of them

struct BigSync {
  uint64_t full[kBigStages], empty[kBigStages], tfull[2], tempty[2], done;
  uint64_t sfull[kF8Scales], sempty[kF8Scales];
  uint32_t tmem;
  int abort;
};
constexpr size_t kBigSmem = 1024 + (size_t)kBigStages * kBigStage + kF8Scales * kF8M * 4 +
                            kBigEpi * 32 * kBigRowPitch + sizeof(BigSync);
static_assert(kBigSmem <= 227 * 1024, "shared memory");
static_assert(4 * kBigPitch <= kBigRowPitch, "staged rows");

__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_addr(dst)),
               "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols)
               : "memory");
}
__device__ __forceinline__ void tc_mma_f8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                               uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// Arrives on `bar` of both CTAs once every MMA this thread issued before has completed.
__device__ __forceinline__ void tc_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(smem_addr(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// Tensor copies into this CTA's shared memory that complete on the barrier at
// the cluster address `bar` of either CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const void* tmap, int x, int y,
                                                 uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
      "bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_addr(dst)),
      "l"(tmap), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const void* tmap, int x, int y, int z,
                                                 uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
      "bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_addr(dst)),
      "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// Arrival on either CTA's barrier.  It orders tensor-memory loads (complete,
// and fenced) before the MMAs of whoever waits, no ordinary memory, so it needs
// no release at cluster scope, which costs a memory barrier of about 1500
// clocks (with it, the whole product ran at that pace: 275 us).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// 16 consecutive fp32 columns of this thread's tensor-memory lane (no wait).
__device__ __forceinline__ void tmem_ld16_issue(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_wait_ld16(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// An untiled copy to device memory (addresses and bytes multiples of 16) that
// belongs to this thread's current group; the end of the group; waits until the
// thread's groups have read shared memory, and until they are done.
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
               "r"(smem_addr(src)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void bulk_wait() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
__device__ __forceinline__ uint32_t bf16_pair(float2 v) {
  const __nv_bfloat162 b = __float22bfloat162_rn(v);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// What a pair works on: a tile, or (h 0 or 1) the half of it whose weights are
// rows 64 h .. 64 h + 63 of both CTAs'.  The tiles of a last round that would
// leave half of the pairs idle are given out in halves (256 x 65536 x 2688, 256
// tiles on 74 pairs: 59.2 us in whole ones, 57.5 so).
struct BigTile {
  int tt, nt, h;
};
struct BigTiles {
  int tchunks, whole, units;
  __host__ __device__ BigTiles(int tokens, int rows, int pairs) {
    tchunks = (tokens + 2 * kF8M - 1) / (2 * kF8M);
    const int tiles = tchunks * ((rows + 2 * kF8M - 1) / (2 * kF8M));
    const int rest = tiles % pairs;
    const bool halves = 2 * rest <= pairs;
    whole = halves ? tiles - rest : tiles;
    units = halves ? tiles + rest : tiles;
  }
  __device__ BigTile at(int u) const {
    BigTile t;
    const int i = u < whole ? u : whole + ((u - whole) >> 1);
    t.h = u < whole ? -1 : (u - whole) & 1;
    t.nt = i / tchunks;
    t.tt = i - t.nt * tchunks;
    return t;
  }
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kBigThreads, 1)
    f8_big_kernel(const __grid_constant__ F8Maps maps, const F8Pass p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  float* s_scale = reinterpret_cast<float*>(stages + kBigStages * kBigStage);
  uint8_t* s_out = reinterpret_cast<uint8_t*>(s_scale + kF8Scales * kF8M);
  BigSync* sy = reinterpret_cast<BigSync*>(s_out + kBigEpi * 32 * kBigRowPitch);
  volatile int* abort = &sy->abort;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kBigStages; ++s) {
      mbar_init(&sy->full[s], 1);
      mbar_init(&sy->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sy->tfull[b], 1);
      mbar_init(&sy->tempty[b], 2 * kBigEpi);
    }
    for (int s = 0; s < kF8Scales; ++s) {
      mbar_init(&sy->sfull[s], 1);
      mbar_init(&sy->sempty[s], kBigEpi);
    }
    mbar_init(&sy->done, 1);
    sy->abort = 0;
    fence_mbar_init();
  }
  if (warp == kBigEpi + 1) tmem_alloc_pair(&sy->tmem, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sy->tmem, 0);
  griddep_wait();
  griddep_launch();
  const int tile0 = (int)blockIdx.x >> 1, tstep = (int)gridDim.x >> 1;
  const BigTiles tiles(p.tokens, p.rows, p.pairs);
  const int ntiles = tiles.units;

  if (warp == kBigEpi) {  // ------------------------------- producer
    const bool one = elect_one();
    RingPos rp, sp;
    int q = 0;
    bool ok = true;
    for (int tile = tile0; tile < ntiles && ok; tile += tstep) {
      const BigTile u = tiles.at(tile);
      const int t0 = u.tt * 2 * kF8M + (int)rank * kF8M, n0 = u.nt * 2 * kF8M + (int)rank * kF8M;
      const uint32_t sbytes = (uint32_t)max(0L, min((long)kF8M, p.xs_pitch - t0)) * 4u;
      for (int kb = 0; kb < p.kblocks; ++kb) {
        ok = (q < kBigStages || f8_wait_warp(&sy->empty[rp.s], rp.phase ^ 1u, p.status, abort)) &&
             (q < kF8Scales || f8_wait_warp(&sy->sempty[sp.s], sp.phase ^ 1u, p.status, abort));
        if (!ok) break;
        uint8_t* st = stages + rp.s * kBigStage;
        // both CTAs' copies complete on the first one's barrier
        const uint32_t bar = cluster_map(&sy->full[rp.s], 0);
        if (one) {
          if (rank == 0) mbar_expect_tx(&sy->full[rp.s], 2 * kBigStage);
          tma_load_2d_pair(st, &maps.x, kb * kF8Block, t0, bar);
          tma_load_3d_pair(st + kF8M * kF8Block, &maps.w0, kb * kF8Block, n0, 0, bar);
          mbar_expect_tx(&sy->sfull[sp.s], sbytes);
          if (sbytes)
            tma_load_1d(s_scale + sp.s * kF8M, p.xs + (long)kb * p.xs_pitch + t0, sbytes,
                        &sy->sfull[sp.s]);
        }
        ++q;
        rp.next(kBigStages);
        sp.next(kF8Scales);
      }
    }
    __syncwarp();
  } else if (warp == kBigEpi + 1) {  // -------------------------- MMA
    const bool one = elect_one();
    if (rank == 0) {
      RingPos rp, ap;
      int q = 0;
      bool ok = true;
      const uint64_t desc = sw128_desc(stages);
      for (int tile = tile0; tile < ntiles && ok; tile += tstep) {
        const BigTile u = tiles.at(tile);
        const uint32_t idesc =
            (1u << 4) | ((u.h < 0 ? 256u >> 3 : 128u >> 3) << 17) | ((256u >> 4) << 24);
        const uint32_t boff = (kF8M * kF8Block >> 4) + (u.h > 0 ? 64 * kF8Block >> 4 : 0);
        for (int kb = 0; kb < p.kblocks; ++kb) {
          ok = (q < 2 || f8_wait_warp(&sy->tempty[ap.s], ap.phase ^ 1u, p.status, abort)) &&
               f8_wait_warp(&sy->full[rp.s], rp.phase, p.status, abort);
          if (!ok) break;
          tc_fence_after();
          const uint64_t ad = desc + (uint32_t)rp.s * (kBigStage >> 4);
          const uint64_t bd = ad + boff;
          if (one) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              tc_mma_f8_pair(tmem + ap.s * 256, ad + 2 * j, bd + 2 * j, idesc, j != 0);
            tc_commit_pair(&sy->empty[rp.s]);
            tc_commit_pair(&sy->tfull[ap.s]);
          }
          __syncwarp();
          ++q;
          rp.next(kBigStages);
          ap.next(2);
        }
      }
      // every MMA issued has completed before shared and tensor memory go
      if (one) tc_commit_pair(&sy->done);
    }
    mbar_wait(&sy->done, 0, nullptr);
    __syncwarp();
  } else {  // -------------------------------------------------- epilogue
    const int quad = warp & 3, part = warp >> 2;
    const uint32_t lane_base = (uint32_t)(32 * quad) << 16;
    uint8_t* staged = s_out + warp * 32 * kBigRowPitch;  // this warp's
    uint32_t* so = reinterpret_cast<uint32_t*>(staged);
    uint4* mine = reinterpret_cast<uint4*>(staged + lane * kBigRowPitch);
    const int size = p.out_bf16 ? 2 : 4;  // bytes of an output value
    const bool bulk = p.ldo * size % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
    const bool words = p.ldo % 2 == 0 && reinterpret_cast<uintptr_t>(p.out) % 4 == 0;
    RingPos ap, sp;
    bool ok = true;
    for (int tile = tile0; tile < ntiles && ok; tile += tstep) {
      const BigTile u = tiles.at(tile);
      const int t0 = u.tt * 2 * kF8M + (int)rank * kF8M + 32 * quad;  // this warp's first token
      // its first column; of a half, the first two parts have 64 columns each
      const int n0 = u.nt * 2 * kF8M + (u.h < 0 ? part * 64 : (part & 1) * kF8M + u.h * 64);
      const bool idle = u.h >= 0 && part >= 2;
      const float* ws = p.ws0 + (long)min(n0 / kF8M, p.rblocks - 1) * p.kblocks;
      float2 acc[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) acc[c] = make_float2(0.0f, 0.0f);
      float wl = 0.0f;
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if ((kb & 31) == 0) wl = kb + lane < p.kblocks ? __ldg(ws + kb + lane) : 0.0f;
        ok = f8_wait(&sy->sfull[sp.s], sp.phase, p.status, abort);
        const float f = s_scale[sp.s * kF8M + 32 * quad + lane] * __shfl_sync(0xffffffffu, wl, kb & 31);
        ok = ok && f8_wait(&sy->tfull[ap.s], ap.phase, p.status, abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t from = tmem + lane_base + ap.s * 256 + part * 64;
        const float2 f2 = make_float2(f, f);
        if (idle) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive_cluster(cluster_map(&sy->tempty[ap.s], 0));
            mbar_arrive(&sy->sempty[sp.s]);
          }
          ap.next(2);
          sp.next(kF8Scales);
          continue;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // 16 columns
          uint32_t d[16];
          tmem_ld16_issue(from + 16 * i, d);
          tmem_wait_ld16(d);
          if (i == 3) {  // everything read: the buffer and the scales are free
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive_cluster(cluster_map(&sy->tempty[ap.s], 0));
              mbar_arrive(&sy->sempty[sp.s]);
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            acc[8 * i + j] =
                __ffma2_rn(make_float2(__uint_as_float(d[2 * j]), __uint_as_float(d[2 * j + 1])), f2,
                           acc[8 * i + j]);
        }
        ap.next(2);
        sp.next(kF8Scales);
      }
      if (!ok) break;
      if (idle) continue;
      bulk_wait_read();  // the rows staged before have left
      if (bulk && n0 + 64 <= p.rows) {
        // every lane stages its token's 64 values and has them copied, while the
        // next tile goes on (fp32: 32 values twice).  That takes the room of a
        // fifth stage of operands.  1024 x 8192 x 512 bf16 20.5 -> 18.6 us, 2048 x
        // 14336 x 4096 133 -> 129 (fp32 147 -> 141), 512 x 14336 x 8192 78.7 -> 79.4;
        // five stages and half the room 137.  Tensor copies, a warp's or by one
        // warp for all, gained no more.  (Each pair of figures is of one run; the
        // clock moves them by a few per cent between runs.)
        uint8_t* o = static_cast<uint8_t*>(p.out) + ((long)(t0 + lane) * p.ldo + n0) * size;
        const bool valid = t0 + lane < p.tokens;
        if (p.out_bf16) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            mine[j] = make_uint4(bf16_pair(acc[4 * j]), bf16_pair(acc[4 * j + 1]),
                                 bf16_pair(acc[4 * j + 2]), bf16_pair(acc[4 * j + 3]));
          fence_proxy_async_smem();
          if (valid) bulk_store(o, mine, kBigRow);
          bulk_commit();
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h) bulk_wait_read();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 a = acc[16 * h + 2 * j], b = acc[16 * h + 2 * j + 1];
              mine[j] = make_uint4(__float_as_uint(a.x), __float_as_uint(a.y),
                                   __float_as_uint(b.x), __float_as_uint(b.y));
            }
            fence_proxy_async_smem();
            if (valid) bulk_store(o + h * kBigRow, mine, kBigRow);
            bulk_commit();
          }
        }
        continue;
      }
      __syncwarp();  // every lane's rows have
      // to row-major through shared memory: 16 words of the warp's 32 rows at a
      // time, stored two rows an instruction
      const int r2 = lane >> 4, w = lane & 15;
      if (p.out_bf16) {
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 32 columns, two a word
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const __nv_bfloat162 v = __float22bfloat162_rn(acc[16 * h + j]);
            so[lane * kBigPitch + j] = *reinterpret_cast<const uint32_t*>(&v);
          }
          __syncwarp();
          const int n = n0 + 32 * h + 2 * w;
#pragma unroll 8
          for (int i = 0; i < 32; i += 2) {
            const uint32_t v = so[(i + r2) * kBigPitch + w];
            if (t0 + i + r2 >= p.tokens) continue;
            __nv_bfloat16* o = out + (long)(t0 + i + r2) * p.ldo + n;
            if (words && n + 1 < p.rows) {
              *reinterpret_cast<uint32_t*>(o) = v;
            } else {
              const __nv_bfloat162 b = *reinterpret_cast<const __nv_bfloat162*>(&v);
              if (n < p.rows) o[0] = b.x;
              if (n + 1 < p.rows) o[1] = b.y;
            }
          }
          __syncwarp();
        }
      } else {
        float* out = static_cast<float*>(p.out);
#pragma unroll
        for (int h = 0; h < 4; ++h) {  // 16 columns
#pragma unroll
          for (int j = 0; j < 16; ++j)
            so[lane * kBigPitch + j] =
                __float_as_uint(j & 1 ? acc[8 * h + j / 2].y : acc[8 * h + j / 2].x);
          __syncwarp();
          const int n = n0 + 16 * h + w;
#pragma unroll 8
          for (int i = 0; i < 32; i += 2) {
            const uint32_t v = so[(i + r2) * kBigPitch + w];
            if (t0 + i + r2 < p.tokens && n < p.rows)
              out[(long)(t0 + i + r2) * p.ldo + n] = __uint_as_float(v);
          }
          __syncwarp();
        }
      }
    }
    bulk_wait();
  }
  if (*abort) f8_linger();
  __syncwarp();
  tc_fence_before();
  cluster_sync();  // neither CTA's shared or tensor memory is in use any more
  if (warp == kBigEpi + 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ------------------------------------------------------------ experts

// One CTA: groups the entries (token t, rank j; id t * k + j) by expert:
// entry i's row is row_start[expert] + pos[i].  Every expert's rows start at a
// multiple of 4 (the scales' bulk copies start on 16 bytes); chunks of at most
// nt rows go to tiles in expert order.  Entries whose expert is outside [0, E)
// are in no group.  The order within an expert follows arrival and changes no
// value: every row is computed alone.
__global__ void __launch_bounds__(1024) f8_plan_kernel(const int* __restrict__ sel, int n, int E,
                                                       int nt, int* pos, int* row_start,
                                                       int4* tiles, int* nchunks) {
  constexpr int kPer = 8;  // entries of a thread whose loads are in flight together
  __shared__ int s_count[1024], s_warp[2][32];
  griddep_wait();
  griddep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  s_count[tid] = 0;
  __syncthreads();
  for (int i0 = tid; i0 < n; i0 += 1024 * kPer) {
    int e[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) e[j] = i0 + 1024 * j < n ? sel[i0 + 1024 * j] : -1;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (e[j] >= 0 && e[j] < E) pos[i0 + 1024 * j] = atomicAdd(&s_count[e[j]], 1);
  }
  __syncthreads();
  const int cnt = s_count[tid], pad = (cnt + 3) & ~3, ch = (cnt + nt - 1) / nt;
  int a = pad, b = ch;  // inclusive scans over the experts
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int va = __shfl_up_sync(0xffffffffu, a, o), vb = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) a += va, b += vb;
  }
  if (lane == 31) s_warp[0][warp] = a, s_warp[1][warp] = b;
  __syncthreads();
  if (warp == 0) {
    int va = s_warp[0][lane], vb = s_warp[1][lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int wa = __shfl_up_sync(0xffffffffu, va, o), wb = __shfl_up_sync(0xffffffffu, vb, o);
      if (lane >= o) va += wa, vb += wb;
    }
    s_warp[0][lane] = va, s_warp[1][lane] = vb;
  }
  __syncthreads();
  const int row = a - pad + (warp ? s_warp[0][warp - 1] : 0);
  const int chunk = b - ch + (warp ? s_warp[1][warp - 1] : 0);
  if (tid < E) row_start[tid] = row;
  for (int c = 0; c < ch; ++c)
    tiles[chunk + c] = make_int4(row + c * nt, min(nt, cnt - c * nt), tid, 0);
  if (tid == 1023) *nchunks = s_warp[1][31];
}

// out[t] = sum over ranks j, in order, of weight * partial row.  Four columns a
// thread.
__global__ void __launch_bounds__(256) f8_combine_kernel(const float* partial, long ldp,
                                                         const int* sel, int E,
                                                         const float* weights, int k, int cols,
                                                         void* out, long ldo, int out_bf16) {
  griddep_wait();
  griddep_launch();
  const long t = blockIdx.x;
  for (int c = (blockIdx.y * 256 + threadIdx.x) * 4; c < cols; c += gridDim.y * 1024) {
    float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int j = 0; j < k; ++j) {
      const int e = sel[t * k + j];
      if (e >= 0 && e < E) {
        const float w = weights[t * k + j];
        const float4 v = __ldcg(reinterpret_cast<const float4*>(partial + (t * k + j) * ldp + c));
        a[0] = fmaf(w, v.x, a[0]), a[1] = fmaf(w, v.y, a[1]);
        a[2] = fmaf(w, v.z, a[2]), a[3] = fmaf(w, v.w, a[3]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < cols) store_out(out, out_bf16, t * ldo + c + i, a[i]);
  }
}

__global__ void f8_check_scales_kernel(const float* s, size_t n, unsigned* bad) {
  unsigned c = 0;
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n;
       i += (size_t)gridDim.x * blockDim.x)
    c += !isfinite(s[i]);
  if (c) atomicAdd(bad, c);
}

// ------------------------------------------------------------ host side

PFN_cuTensorMapEncodeTiled_v12000 f8_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault,
                                         &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  return encode;
}

bool f8_encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims,
               const cuuint64_t* strides, int box_rows) {
  const auto encode = f8_encoder();
  if (!encode) return false;
  const cuuint32_t box[3] = {(cuuint32_t)kF8Block, (cuuint32_t)box_rows, 1}, elem[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides,
                box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Weights as [experts][rows][cols] bytes, a tile's box 128 x 128; what lies
// past the rows or columns of an expert reads as zeros.
bool f8_weight_map(CUtensorMap* map, const F8Matrix& w) {
  const cuuint64_t dims[3] = {(cuuint64_t)w.cols, (cuuint64_t)w.rows, (cuuint64_t)w.experts};
  const cuuint64_t strides[2] = {(cuuint64_t)w.pitch, (cuuint64_t)w.pitch * w.rows};
  return f8_encode(map, w.data, 3, dims, strides, kF8M);
}

bool f8_rows_map(CUtensorMap* map, const void* q, long pitch, long rows, int cols, int nt) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  return f8_encode(map, q, 2, dims, strides, nt);
}

constexpr long kF8MaxTiles = 1L << 30;  // tiles are counted in 32 bits

// Raises a kernel's shared-memory limit, once per kernel and device.
cudaError_t f8_allow_smem(const void* kern, size_t bytes) {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  if (done.count({kern, dev})) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done.insert({kern, dev});
  return e;
}

// CTAs to a tile.  Where the tiles (an upper bound of them) leave multiprocessors
// idle, clusters share a tile's K as long as every CTA has one to itself and a few blocks of K.  One
// token, cold: 512 rows of 8192 columns 22.5 us unsplit, 12.6 in eight; 4096 of
// 4096 17.3, 14.5 in four; 2688 of 1856 12.5, 12.3 in four; 14336 of 4096 (112
// tiles) 22.5 unsplit, and with 24 tokens 22.6 against 26.7 in two.
int f8_split(long tiles, int kblocks) {
  int split = 1;
  while (split < kF8MaxSplit && tiles * split * 2 <= sm_count() &&
         split * 2 * kF8SplitBlocks <= kblocks)
    split *= 2;
  return split;
}

template <int NT, int MATS, int MODE>
cudaError_t launch_f8_gemm(const F8Maps& maps, F8Pass p, long tiles, cudaStream_t s) {
  using C = F8Cfg<NT, MATS, MODE>;
  const long slots = (long)sm_count() * C::kCtas;
  if (tiles > kF8MaxTiles) return cudaErrorInvalidValue;
  p.split = f8_split(tiles, p.kblocks);
  auto kern = p.split > 1 ? f8_gemm_kernel<NT, MATS, MODE, true>
                          : f8_gemm_kernel<NT, MATS, MODE, false>;
  const cudaError_t e = f8_allow_smem(reinterpret_cast<const void*>(kern), C::kSmem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.split > 1 || C::kGroup ? tiles * p.split
                                                                  : std::min(tiles, slots)));
  cfg.blockDim = dim3(kF8Threads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = p.split;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, maps, p);
}

template <int MATS, int MODE>
cudaError_t launch_f8_pass(int nt, const F8Maps& maps, const F8Pass& p, long tiles,
                           cudaStream_t s) {
  switch (nt) {
    case 16: return launch_f8_gemm<16, MATS, MODE>(maps, p, tiles, s);
    case 32: return launch_f8_gemm<32, MATS, MODE>(maps, p, tiles, s);
    default: return launch_f8_gemm<64, MATS, MODE>(maps, p, tiles, s);
  }
}

// Rows of x in a tile of the small kind: as few columns as hold the tokens, 64
// at most.  (Columns of 128 leave the weights half as many trips from L2, but
// one CTA a multiprocessor instead of two: 2048 tokens, 2 of 8 experts of 2048 x
// 1856 with gate 240 us, in 64 159; 128 tokens by 2688 x 8192 41 us and 31.)
int f8_chunk(long rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

int f8_blocks(long n) { return (int)((n + kF8Block - 1) / kF8Block); }

template <typename T>
cudaError_t quant_t(const T* x, long ldx, int tokens, int cols, uint8_t* q, long q_pitch,
                    float* scales, long s_pitch, const F8Rows& rows, cudaStream_t st) {
  const int vec = ldx % 4 == 0 && reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0;
  const long per = (f8_blocks(cols) + kQuantBlocks - 1) / kQuantBlocks;
  const long units = (rows.sel ? (long)tokens : s_pitch) * per;
  if (units > 0x3fffffffL) return cudaErrorInvalidValue;
  const long ctas = (units + 7) / 8;
  auto kern = rows.sel ? f8_quant_kernel<T, true> : f8_quant_kernel<T, false>;
  return launch_pdl(kern, dim3((unsigned)ctas), dim3(256), 0, st, x, ldx, tokens, cols, q,
                    (int)q_pitch, scales, (int)s_pitch, rows, vec);
}

cudaError_t quant(bool bf16, const void* x, long ldx, int tokens, int cols, uint8_t* q,
                  long q_pitch, float* scales, long s_pitch, const F8Rows& rows, cudaStream_t st) {
  return bf16 ? quant_t(static_cast<const __nv_bfloat16*>(x), ldx, tokens, cols, q, q_pitch,
                        scales, s_pitch, rows, st)
              : quant_t(static_cast<const float*>(x), ldx, tokens, cols, q, q_pitch, scales,
                        s_pitch, rows, st);
}

}  // namespace

cudaError_t launch_f8_quant(bool bf16, const void* x, long ldx, int tokens, int cols, uint8_t* q,
                            float* scales, cudaStream_t st) {
  return quant(bf16, x, ldx, tokens, cols, q, f8_pad16(cols), scales, f8_pad4(tokens), F8Rows{}, st);
}

cudaError_t f8_check_scales(const float* scales, size_t n, unsigned* bad, cudaStream_t st) {
  f8_check_scales_kernel<<<(unsigned)std::min<size_t>((n + 255) / 256, 1024), 256, 0, st>>>(
      scales, n, bad);
  return cudaGetLastError();
}

cudaError_t f8_prepare(F8Matrix* w) {
  return f8_weight_map(&w->map, *w) ? cudaSuccess : cudaErrorInvalidValue;
}

// Rows of x that four consecutive values can be loaded from at once.
static bool f8_rows_vec(bool bf16, const void* x, long ldx, int tokens) {
  return (tokens == 1 || ldx % 4 == 0) && reinterpret_cast<uintptr_t>(x) % (bf16 ? 8 : 16) == 0;
}

// One launch and no workspace against two, for what every CTA does over again.
// By 4096 x 4096 (8 blocks a CTA) 24 tokens, 48 pairs, take 12.0 us and 15.4 in
// two launches; by 14336 x 4096 (32 blocks) 8 tokens, 64 pairs, 17.9 and 15.0.
bool f8_step_applies(const F8Matrix& w, int tokens) {
  const int nt = f8_chunk(tokens), kb = f8_blocks(w.cols);
  if (tokens > kF8StepTokens) return false;
  const int split = f8_split(f8_blocks(w.rows), kb), most = (kb + split - 1) / split;
  const int room =
      nt == 16 ? F8Cfg<16, 1, kF8Step>::kStepBlocks : F8Cfg<32, 1, kF8Step>::kStepBlocks;
  return most <= room &&
         tokens * ((most + kQuantBlocks - 1) / kQuantBlocks) <= kF8StepMost;
}

cudaError_t launch_f8_step(const F8Matrix& w, bool x_bf16, const void* x, long ldx, int tokens,
                           bool out_bf16, void* out, long ldo, int* status, cudaStream_t st) {
  F8Maps maps;
  maps.x = maps.w0 = maps.w1 = w.map;
  F8Pass p{};
  p.rows = w.rows;
  p.rblocks = f8_blocks(w.rows);
  p.kblocks = f8_blocks(w.cols);
  p.ws0 = w.scales;
  p.tokens = tokens;
  p.chunks = 1;
  p.x = x;
  p.ldx = ldx;
  p.cols = w.cols;
  p.x_bf16 = x_bf16;
  p.x_vec = f8_rows_vec(x_bf16, x, ldx, tokens);
  p.out = out;
  p.ldo = ldo;
  p.out_bf16 = out_bf16;
  p.status = status;
  return f8_chunk(tokens) == 16 ? launch_f8_gemm<16, 1, kF8Step>(maps, p, p.rblocks, st)
                                : launch_f8_gemm<32, 1, kF8Step>(maps, p, p.rblocks, st);
}

cudaError_t launch_f8_project(const F8Matrix& w, const uint8_t* q, const float* scales, int tokens,
                              bool out_bf16, void* out, long ldo, bool after_quant, int* status,
                              cudaStream_t st) {
  F8Maps maps;
  // Pairs where the small tiles would come in several rounds.  Small and pairs:
  // 256 tokens by 4096 x 8192 (128 small tiles) 38 and 41 us, 512 by 1024 x 8192
  // (64) 34 and 41, by 2688 x 8192 (168) 49 and 44, by 14336 x 8192 (896) 145
  // and 80.
  const int nt_small = f8_chunk(tokens);
  const bool big = tokens > nt_small && (long)f8_blocks(w.rows) *
                                                ((tokens + nt_small - 1) / nt_small) > sm_count();
  const int nt = big ? kF8M : nt_small;
  maps.w0 = maps.w1 = w.map;
  if (!f8_rows_map(&maps.x, q, f8_pad16(w.cols), tokens, w.cols, nt)) return cudaErrorInvalidValue;
  F8Pass p{};
  p.rows = w.rows;
  p.rblocks = f8_blocks(w.rows);
  p.kblocks = f8_blocks(w.cols);
  p.ws0 = w.scales;
  p.xs = scales;
  p.xs_pitch = f8_pad4(tokens);
  p.tokens = tokens;
  p.chunks = (tokens + nt - 1) / nt;
  p.out = out;
  p.ldo = ldo;
  p.out_bf16 = out_bf16;
  p.early = after_quant;
  p.status = status;
  if (!big) return launch_f8_pass<1, kF8Out>(nt, maps, p, (long)p.chunks * p.rblocks, st);
  const cudaError_t e = f8_allow_smem(reinterpret_cast<const void*>(f8_big_kernel), kBigSmem);
  if (e != cudaSuccess) return e;
  if ((long)((tokens + 255) / 256) * ((w.rows + 255) / 256) > kF8MaxTiles)
    return cudaErrorInvalidValue;
  p.pairs = sm_count() / 2;
  const int units = BigTiles(tokens, w.rows, p.pairs).units;
  return launch_pdl(f8_big_kernel, dim3((unsigned)(2 * std::min(units, p.pairs))),
                    dim3(kBigThreads), kBigSmem, st, maps, p);
}

F8MoeLayout f8_moe_layout(const F8Moe& m, long tokens, int k) {
  F8MoeLayout L;
  const long n = tokens * k, groups = std::min<long>(n, m.up.experts);
  L.rows = f8_pad4(n + 3 * groups);
  L.max_chunks = n / 16 + groups;
  auto take = [off = size_t(0)](size_t bytes) mutable {
    const size_t at = off;
    off += (bytes + 255) & ~size_t(255);
    return at;
  };
  L.hp = (long)f8_blocks(m.up.rows) * kF8Block;
  L.pos = take((size_t)n * 4);
  L.row_start = take((size_t)m.up.experts * 4);
  L.entry = take((size_t)L.rows * 4);
  L.tiles = take((size_t)L.max_chunks * 16);
  L.nchunks = take(4);
  L.counters = take((size_t)f8_blocks(m.down.rows) * 4);
  L.xq = take((size_t)L.rows * f8_pad16(m.up.cols));
  L.xs = take((size_t)f8_blocks(m.up.cols) * L.rows * 4);
  L.hq = take((size_t)L.rows * L.hp);
  L.hs = take((size_t)f8_blocks(m.up.rows) * L.rows * 4);
  L.ldp = f8_pad4(m.down.rows);
  L.partial = take((size_t)n * L.ldp * 4);
  L.bytes = take(0);
  return L;
}

cudaError_t launch_f8_moe(const F8Moe& m, bool x_bf16, const void* x, long ldx, int tokens, int k,
                          const int* sel, const float* weights, bool out_bf16, void* out, long ldo,
                          void* work, int* status, cudaStream_t st) {
  const F8MoeLayout L = f8_moe_layout(m, tokens, k);
  uint8_t* base = static_cast<uint8_t*>(work);
  int* pos = reinterpret_cast<int*>(base + L.pos);
  int* row_start = reinterpret_cast<int*>(base + L.row_start);
  int* entry = reinterpret_cast<int*>(base + L.entry);
  int4* tiles = reinterpret_cast<int4*>(base + L.tiles);
  int* nchunks = reinterpret_cast<int*>(base + L.nchunks);
  float* partial = reinterpret_cast<float*>(base + L.partial);
  const long n = (long)tokens * k;
  // chunks of an expert's tokens: half again the average, so most experts take one
  const int nt = f8_chunk((3 * n / std::min<long>(n, m.up.experts) + 1) / 2);
  const long chunks = n / nt + std::min<long>(n, m.up.experts);
  // A call so small that the down product has one tile a CTA at most takes two
  // launches instead of five: every CTA of the gate and up product groups the
  // entries and quantises its rows for itself, and the down product's CTAs add
  // the entries up (one token, 10 of 512 experts: 18 us against 31).  With more tiles the
  // fence after each, and the weights that the plan's own launch lets the gate
  // and up product request ahead, cost more (32 tokens, 6 of 128 experts of 2688 x
  // 1856: 215 us against 157).  Its CTAs hold kStepBlocks blocks of K: wider layers
  // whose K is not shared (H above 2688) take five launches at one token too.
  const int kb_up = f8_blocks(m.up.cols), rb_up = f8_blocks(m.up.rows);
  const int split_up = f8_split(chunks * rb_up, kb_up);
  const bool few = n <= kF8StepEntries && nt == 16 &&
                   (kb_up + split_up - 1) / split_up <=
                       (m.gate.data ? F8Cfg<16, 2, kF8StepAct>::kStepBlocks
                                    : F8Cfg<16, 1, kF8StepAct>::kStepBlocks) &&
                   chunks * f8_blocks(m.down.rows) <=
                       (long)sm_count() * F8Cfg<16, 1, kF8StepPartial>::kCtas;
  int* counters = few ? reinterpret_cast<int*>(base + L.counters) : nullptr;
  cudaError_t e = cudaSuccess;
  if (!few) {
    e = launch_pdl(f8_plan_kernel, dim3(1), dim3(1024), 0, st, sel, (int)n, m.up.experts, nt, pos,
                   row_start, tiles, nchunks);
    if (e != cudaSuccess) return e;
    const F8Rows rows{sel, pos, row_start, entry, k, m.up.experts};
    e = quant(x_bf16, x, ldx, tokens, m.up.cols, base + L.xq, f8_pad16(m.up.cols),
              reinterpret_cast<float*>(base + L.xs), L.rows, rows, st);
    if (e != cudaSuccess) return e;
  }
  F8Maps maps;
  F8Pass p{};
  maps.w0 = m.gate.data ? m.gate.map : m.up.map;
  maps.w1 = m.up.map;
  maps.x = maps.w1;  // not used by few entries' kernel
  if (!few && !f8_rows_map(&maps.x, base + L.xq, f8_pad16(m.up.cols), L.rows, m.up.cols, nt))
    return cudaErrorInvalidValue;
  p.rows = m.up.rows;
  p.rblocks = f8_blocks(m.up.rows);
  p.kblocks = f8_blocks(m.up.cols);
  p.ws0 = m.gate.data ? m.gate.scales : m.up.scales;
  p.ws1 = m.up.scales;
  p.xs = reinterpret_cast<const float*>(base + L.xs);
  p.xs_pitch = L.rows;
  p.tiles = tiles;
  p.nchunks = nchunks;
  p.hq = base + L.hq;
  p.h_pitch = L.hp;
  p.hs = reinterpret_cast<float*>(base + L.hs);
  p.hs_pitch = L.rows;
  p.early = 1;
  p.status = status;
  if (few) {
    p.early = 0;
    p.tiles = nullptr;
    p.x = x;
    p.ldx = ldx;
    p.cols = m.up.cols;
    p.x_bf16 = x_bf16;
    p.x_vec = f8_rows_vec(x_bf16, x, ldx, tokens);
    p.sel = sel;
    p.k = k;
    p.E = m.up.experts;
    p.n = (int)n;
    p.counters = counters;
    p.nclear = f8_blocks(m.down.rows);
    // one CTA (or cluster) a tile: a CTA quantises the rows of one
    e = m.gate.data ? launch_f8_gemm<16, 2, kF8StepAct>(maps, p, chunks * p.rblocks, st)
                    : launch_f8_gemm<16, 1, kF8StepAct>(maps, p, chunks * p.rblocks, st);
  } else {
    e = m.gate.data ? launch_f8_pass<2, kF8Act>(nt, maps, p, chunks * p.rblocks, st)
                    : launch_f8_pass<1, kF8Act>(nt, maps, p, chunks * p.rblocks, st);
  }
  if (e != cudaSuccess) return e;
  F8Pass d{};
  maps.w0 = maps.w1 = m.down.map;
  if (!f8_rows_map(&maps.x, base + L.hq, L.hp, L.rows, m.down.cols, nt))
    return cudaErrorInvalidValue;
  d.rows = m.down.rows;
  d.rblocks = f8_blocks(m.down.rows);
  d.kblocks = f8_blocks(m.down.cols);
  d.ws0 = m.down.scales;
  d.xs = p.hs;
  d.xs_pitch = L.rows;
  d.tiles = tiles;
  d.nchunks = nchunks;
  d.partial = partial;
  d.ldp = L.ldp;
  d.entry = entry;
  d.early = 1;
  d.status = status;
  if (few) {
    d.tiles = nullptr;
    d.n = (int)n;
    d.counters = counters;
    d.sel = sel;
    d.weights = weights;
    d.k = k;
    d.E = m.up.experts;
    d.tokens = tokens;
    d.out = out;
    d.ldo = ldo;
    d.out_bf16 = out_bf16;
    return launch_f8_gemm<16, 1, kF8StepPartial>(maps, d, chunks * d.rblocks, st);
  }
  e = launch_f8_pass<1, kF8Partial>(nt, maps, d, chunks * d.rblocks, st);
  if (e != cudaSuccess) return e;
  const unsigned gy = (unsigned)std::max(1, std::min((m.down.rows + 1023) / 1024, 64));
  return launch_pdl(f8_combine_kernel, dim3((unsigned)tokens, gy), dim3(256), 0, st, partial,
                    L.ldp, sel, m.up.experts, weights, k, m.down.rows, out, ldo, (int)out_bf16);
}

}  // namespace lb
