// Attention of one new token per sequence over a paged cache, split over the cache's length and joined.
//
//   s_j = scale q.k_j  (capped: c tanh(s_j / c)),   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   lse = m + log sum
//
// A key and a value are read once and used by the 1 - 16 query heads that share them, so memory bounds the kernel: about 23
// bytes a cycle and SM have to arrive, and the arithmetic only has to keep up. The products run on warp-level matrix
// instructions with the KEYS as the tile's 16 rows and the query heads as its 8 columns: a group of up to eight heads
// wastes nothing (with the heads as rows, half and more of each instruction would be padding), and 16 keys a warp are
// enough to feed it. tcgen05 needs 128 rows to a tile and accumulators in TMEM; it has nothing to give where the tensor pipe idles.
//
//   S^T [16 keys, 8 heads] = K [16, D] Q^T [D, 8]          A = K rows as they lie, B = queries, kept in registers
//   O^T [D, 8 heads]      += V^T [D, 16 keys] P^T [16, 8]  A = V transposed on the way out of shared memory
//
// The accumulator layout of S^T differs from the operand layout of P^T by a transposition of 8 x 8 blocks (movmatrix).
// Both products have a head's values in the same lanes, so rescaling O by the change of the maximum needs no exchange.
//
// Each warp streams keys of its own through a ring of stages (cp.async; rows behind the end, of bad pages and before the
// window arrive as zeros and score -inf), with a running maximum and sum of its own: no barrier until the pair is done. Then the
// block's four warps are joined through shared memory. Blocks take equal shares of the line of all tiles (attention_plan.hpp); a pair that several
// blocks share leaves unnormalised partial results, which join_kernel adds in the order of the blocks: results
// do not depend on which block is done first.
//
// e4m3 caches: codes become fp16 exactly (cvt), a key's factor multiplies its score, a value's factor its probability.
#include "attention_common.cuh"

#include <atomic>

namespace rocshmem {
namespace kernels {

namespace attn {
namespace {

constexpr int kWarps = 4;
constexpr int kPagedThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Probabilities are at most 1. Where they are rounded to fp16 they are scaled by 2^14 first, so that one down to 2^-28 of
// the largest keeps all its bits and none above 2^-39 is lost from a long sum; the factor is in the sum as well and cancels.
constexpr float kF16Shift = 14.f;

enum Mode : int { MODE_BF16 = 0, MODE_F16 = 1, MODE_E4M3 = 2 };

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <bool BF16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// Two e4m3 codes in the low or high half of `w` as two fp16 values (exact).
__device__ __forceinline__ uint32_t e4m3_lo(uint32_t w) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3);
  return static_cast<uint32_t>(h.x) | static_cast<uint32_t>(h.y) << 16;
}
__device__ __forceinline__ uint32_t e4m3_hi(uint32_t w) { return e4m3_lo(w >> 16); }

// Shared memory and tile sizes of one instantiation. Rows are padded so that the accesses of a fragment fall into
// different banks: 16 bytes for 16-bit rows (ldmatrix), for e4m3 32 bytes a key row (8 bytes a lane from four rows) and 16 a value row
// (up to 16 bytes a lane from every other row). With 96 e4m3 elements a key row already has that stride.
template <int D, int NT, int MODE>
struct Shape {
  static constexpr int kElem = MODE == MODE_E4M3 ? 1 : 2;
  static constexpr int kKeys = D * kElem <= 128 ? 32 : 16;  // keys a warp takes a step
  static constexpr int kTileKeys = kWarps * kKeys;
  static constexpr int kRowBytes = D * kElem;
  static constexpr int kPitchK = kRowBytes + (MODE == MODE_E4M3 ? (D == 96 ? 0 : 32) : 16);
  static constexpr int kPitchV = kRowBytes + 16;
  static constexpr int kScales = MODE == MODE_E4M3 ? 2 * kKeys * 4 : 0;
  static constexpr int kStage = kKeys * (kPitchK + kPitchV) + kScales;  // one warp's stage
  static constexpr int kHeads = 8 * NT;
  // Joining the warps: their maxima and sums, and their accumulators a half of the rows of O^T at a time.
  static constexpr int kStats = 3 * kWarps * kHeads;
  static constexpr int kMerge = (kStats + kWarps * (D / 2) * kHeads) * 4;
  static constexpr int kFixed = kMerge + 16 * kWarps * 4 + 64;
  // Two blocks an SM if three stages or more fit for both, else one block; at most six stages.
  static constexpr int kFitTwo = (113 * 1024 - kFixed) / (kWarps * kStage);
  static constexpr int kFitOne = (226 * 1024 - kFixed) / (kWarps * kStage);
  static constexpr int kBlocks = kFitTwo >= 3 ? 2 : 1;
  static constexpr int kFit = kBlocks == 2 ? kFitTwo : kFitOne;
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kSmem = kFixed + kStages * kWarps * kStage;
  static_assert(kStages >= 3 && kStages <= 16 && kPitchK % 16 == 0 && kPitchV % 16 == 0 && kStage % 16 == 0, "alignment");
};

struct Params {
  const void *q;
  long long q_token, q_head;
  const char *k, *v;
  const float *k_scale, *v_scale;
  const int *table;
  long long table_stride;
  const int *lengths;
  int batch, heads, kv_heads, group, chunks, pages, shift, capacity, window;
  float scale, softcap;
  void *out;
  float *lse;
  int q_bf16, out_f32;
  float *partial;     // [blocks][2][kHeads][D + 2]: unnormalised O, then maximum (base 2) and sum
  long long *bases;   // [batch + 2]: a sequence's first tile; then the total, then tiles per block
  int blocks, least;
};

// Walks the tiles of a block's range in order.
struct Cursor {
  int b, unit, tile, n, first, end;
  int left;  // tiles that remain, this one included
};

__device__ __forceinline__ void enter(Cursor &c, const Params &p, int tile_keys) {
  const Span s = visible(p.lengths[c.b], p.capacity, p.window);
  c.first = s.first;
  c.end = s.end;
  c.n = tiles_of(s, tile_keys);
}

__device__ __forceinline__ void advance(Cursor &c, const Params &p, int tile_keys) {
  if (--c.left <= 0) return;
  if (++c.tile < c.n) return;
  c.tile = 0;
  if (++c.unit < p.kv_heads * p.chunks) return;
  c.unit = 0;
  do {
    ++c.b;
    if (c.b >= p.batch) {  // not reached while tiles remain
      c.left = 0;
      return;
    }
    enter(c, p, tile_keys);
  } while (c.n == 0);
}

template <int D, int NT, int MODE>
__global__ void __launch_bounds__(kPagedThreads, Shape<D, NT, MODE>::kBlocks) paged_kernel(const Params p) {
  using S = Shape<D, NT, MODE>;
  constexpr bool kBf16 = MODE == MODE_BF16;
  constexpr int kKeys = S::kKeys, MT = kKeys / 16, DK = D / 16;
  extern __shared__ __align__(16) char smem[];
  float *stats = reinterpret_cast<float *>(smem + S::kStages * kWarps * S::kStage);
  float *merge = stats + S::kStats;
  uint32_t *masks = reinterpret_cast<uint32_t *>(merge + kWarps * (D / 2) * S::kHeads);  // [stage][warp]
  long long *scan = reinterpret_cast<long long *>(masks + 16 * kWarps);                  // 8 words
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const int units = p.kv_heads * p.chunks;

  // ---- this block's range of the line of tiles ----
  // Threads take neighbouring sequences, `per_thread` each; a scan over the threads gives each one its first tile.
  const int per_thread = (p.batch + kPagedThreads - 1) / kPagedThreads;
  const int b_lo = min(tid * per_thread, p.batch), b_hi = min(b_lo + per_thread, p.batch);
  long long mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += tiles_of(visible(p.lengths[b], p.capacity, p.window), S::kTileKeys);
  mine *= units;
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) upto += scan[w];
    total += scan[w];
  }
  const long long per = per_block(total, p.blocks, p.least);
  const long long t0 = per * blockIdx.x, t1 = min(total, t0 + per);
  // The thread whose sequences hold tile t0 finds the sequence; block 0 writes down all first tiles for the join, and a
  // sequence that sees nothing gets its result here.
  {
    long long at = upto - mine;
    for (int b = b_lo; b < b_hi; ++b) {
      const int n = tiles_of(visible(p.lengths[b], p.capacity, p.window), S::kTileKeys);
      if (t0 < t1 && t0 >= at && t0 < at + static_cast<long long>(n) * units) {
        scan[4] = b;
        scan[5] = t0 - at;
      }
      if (blockIdx.x == 0) p.bases[b] = at;
      at += static_cast<long long>(n) * units;
    }
    if (blockIdx.x == 0 && tid == 0) {
      p.bases[p.batch] = total;
      p.bases[p.batch + 1] = per;
    }
  }
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    const Span s = visible(p.lengths[b], p.capacity, p.window);
    if (s.end > s.first) continue;
    for (int i = tid; i < p.heads * D; i += kPagedThreads) {
      const long long at = static_cast<long long>(b) * p.heads * D + i;
      if (p.out_f32) static_cast<float *>(p.out)[at] = 0.f;
      else static_cast<uint16_t *>(p.out)[at] = 0;
    }
    if (p.lse != nullptr) {
      for (int i = tid; i < p.heads; i += kPagedThreads) p.lse[static_cast<long long>(b) * p.heads + i] = -INFINITY;
    }
  }
  __syncthreads();
  if (t0 >= t1) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    return;
  }
  Cursor cur;
  cur.b = static_cast<int>(scan[4]);
  enter(cur, p, S::kTileKeys);
  cur.unit = static_cast<int>(scan[5] / cur.n);
  cur.tile = static_cast<int>(scan[5] % cur.n);
  cur.left = static_cast<int>(t1 - t0);
  Cursor ahead = cur;

  // ---- loads: `ahead` runs kStages - 1 tiles before `cur`; a tile's page is looked up one step before its rows are ----
  char *const stages = smem + warp * S::kStage;  // a stage of all four warps is kWarps * kStage bytes
  auto look_up = [&](const Cursor &c) -> int {
    if (c.left <= 0) return -1;
    const int pos = c.first + c.tile * S::kTileKeys + warp * kKeys + lane;
    if ((kKeys < 32 && lane >= kKeys) || pos >= c.end) return -1;
    return page_row(p.table[c.b * p.table_stride + (pos >> p.shift)], p.pages, pos, p.shift, p.kv_heads, c.unit / p.chunks);
  };
  auto load = [&](int stage, int row) {
    char *k_s = stages + stage * kWarps * S::kStage, *v_s = k_s + kKeys * S::kPitchK;
    const uint32_t mask = __ballot_sync(0xffffffffu, row >= 0);
    if (lane == 0) masks[stage * kWarps + warp] = mask;
    constexpr int kChunks = S::kRowBytes / 16;
    constexpr int kCopies = kKeys * kChunks / 32;
    static_assert(kKeys * kChunks % 32 == 0, "whole warps");
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int at = i * 32 + lane, r = at / kChunks, c = at % kChunks;
      const int from = __shfl_sync(0xffffffffu, row, r);
      const long long off = from < 0 ? 0 : static_cast<long long>(from) * S::kRowBytes + c * 16;
      const uint32_t bytes = from < 0 ? 0 : 16;
      copy16(smem_addr(k_s + r * S::kPitchK + c * 16), p.k + off, bytes);
      copy16(smem_addr(v_s + r * S::kPitchV + c * 16), p.v + off, bytes);
    }
    if constexpr (MODE == MODE_E4M3) {
      float *s = reinterpret_cast<float *>(v_s + kKeys * S::kPitchV);
      if constexpr (kKeys == 32) {
        copy4(smem_addr(s + lane), p.k_scale + max(row, 0), row < 0 ? 0 : 4);
        copy4(smem_addr(s + kKeys + lane), p.v_scale + max(row, 0), row < 0 ? 0 : 4);
      } else {
        const int from = __shfl_sync(0xffffffffu, row, lane % 16);
        copy4(smem_addr(s + lane), (lane < 16 ? p.k_scale : p.v_scale) + max(from, 0), from < 0 ? 0 : 4);
      }
    }
  };
  int next_row = look_up(ahead);
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) {
    if (ahead.left > 0) {
      load(i, next_row);
      advance(ahead, p, S::kTileKeys);
      next_row = look_up(ahead);
    }
    copies_commit();
  }
  int stage = 0, load_stage = S::kStages - 1;

  // ---- pairs ----
  const int k_lane = (lane % 16) * S::kPitchK + (lane / 16) * 16;                       // ldmatrix: 16 keys x 16 elements
  const int v_lane = ((lane / 16) * 8 + lane % 8) * S::kPitchV + (lane / 8 % 2) * 16;   // transposed
  while (cur.left > 0) {
    const int b = cur.b, kv = cur.unit / p.chunks, h0 = kv * p.group + cur.unit % p.chunks * S::kHeads;
    const int n_heads = min(S::kHeads, (kv + 1) * p.group - h0);
    // Queries as B operands: lane (g, t) has elements of head g. 16-bit caches: 16 kk + 2t, + 1 and + 8, + 9. e4m3:
    // eight neighbouring elements 32 s + 8 t serve two steps, in the order in which the key codes are read.
    uint32_t qf[NT][DK][2];
    float q_scale[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const bool has = 8 * j + g < n_heads;
      const uint16_t *q = static_cast<const uint16_t *>(p.q) + b * p.q_token + (has ? h0 + 8 * j + g : h0) * p.q_head;
      if constexpr (MODE != MODE_E4M3) {
#pragma unroll
        for (int kk = 0; kk < DK; ++kk) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            qf[j][kk][i] = has ? *reinterpret_cast<const uint32_t *>(q + 16 * kk + 8 * i + 2 * t) : 0u;
          }
        }
        q_scale[j][0] = q_scale[j][1] = 1.f;
      } else {
        // A head's largest magnitude brought to [1, 2) by a power of two: bf16 values then fit fp16 exactly, down to
        // 2^-24 of the largest.
        uint4 raw[D / 32];
        uint32_t top = 0;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
          raw[s] = has ? *reinterpret_cast<const uint4 *>(q + 32 * s + 8 * t) : make_uint4(0, 0, 0, 0);
          float x[8];
          if (p.q_bf16) unpack8(Raw8<__nv_bfloat16>{raw[s]}, x);
          else unpack8(Raw8<__half>{raw[s]}, x);
#pragma unroll
          for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^e with e the exponent of the largest, kept where 2^-e is normal too.
        const uint32_t e = min(max(top >> 23, 2u), 252u);
        const float up = __uint_as_float((254u - e) << 23), down = __uint_as_float(e << 23);
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
          float x[8];
          if (p.q_bf16) unpack8(Raw8<__nv_bfloat16>{raw[s]}, x);
          else unpack8(Raw8<__half>{raw[s]}, x);
#pragma unroll
          for (int i = 0; i < 4; ++i) qf[j][2 * s + i / 2][i % 2] = pack2<false>(x[2 * i] * up, x[2 * i + 1] * up);
        }
        // The factors of the heads in this lane's columns, 2t and 2t + 1, lie in lanes 8t and 8t + 4.
        q_scale[j][0] = __shfl_sync(0xffffffffu, down, 8 * t);
        q_scale[j][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) q_scale[j][i] *= p.scale * (p.softcap > 0.f ? 1.f : kLog2e);
    }
    float o[DK][NT][4] = {}, m[NT][2], l[NT][2] = {}, cv = 0x1p-100f;
#pragma unroll
    for (int j = 0; j < NT; ++j) m[j][0] = m[j][1] = -INFINITY;

    const bool begins = cur.tile == 0;
    bool ends = false;
    while (true) {
      copies_wait<S::kStages - 2>();
      __syncwarp();
      if (ahead.left > 0) {
        load(load_stage, next_row);
        advance(ahead, p, S::kTileKeys);
        next_row = look_up(ahead);
      }
      copies_commit();
      load_stage = load_stage + 1 == S::kStages ? 0 : load_stage + 1;

      const char *k_s = stages + stage * kWarps * S::kStage, *v_s = k_s + kKeys * S::kPitchK;
      const float *f_s = reinterpret_cast<const float *>(v_s + kKeys * S::kPitchV);
      const uint32_t mask = masks[stage * kWarps + warp];
      if (mask != 0) {  // a warp may have no key in a pair's last tile
        // S^T
        float s[MT][NT][4] = {};
        if constexpr (MODE != MODE_E4M3) {
#pragma unroll
          for (int kk = 0; kk < DK; ++kk) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              uint32_t a[4];
              ldmatrix4(a, smem_addr(k_s) + i * 16 * S::kPitchK + k_lane + kk * 32);
#pragma unroll
              for (int j = 0; j < NT; ++j) mma<kBf16>(s[i][j], a, qf[j][kk][0], qf[j][kk][1]);
            }
          }
        } else {
#pragma unroll
          for (int ss = 0; ss < D / 32; ++ss) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              const char *at = k_s + (16 * i + g) * S::kPitchK + 32 * ss + 8 * t;
              const uint2 lo = *reinterpret_cast<const uint2 *>(at);
              const uint2 hi = *reinterpret_cast<const uint2 *>(at + 8 * S::kPitchK);
              const uint32_t a0[4] = {e4m3_lo(lo.x), e4m3_lo(hi.x), e4m3_hi(lo.x), e4m3_hi(hi.x)};
              const uint32_t a1[4] = {e4m3_lo(lo.y), e4m3_lo(hi.y), e4m3_hi(lo.y), e4m3_hi(hi.y)};
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                mma<false>(s[i][j], a0, qf[j][2 * ss][0], qf[j][2 * ss][1]);
                mma<false>(s[i][j], a1, qf[j][2 * ss + 1][0], qf[j][2 * ss + 1][1]);
              }
            }
          }
        }
        // Scores in base 2, -inf where there is no key; maxima over the tile.
        float top[NT][2], v_factor[MT][2], v_top = 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j) top[j][0] = top[j][1] = -INFINITY;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int row = 16 * i + 8 * r + g;
            const bool seen = mask >> row & 1;
            float f = 1.f;
            if constexpr (MODE == MODE_E4M3) {
              f = f_s[row];
              v_factor[i][r] = f_s[kKeys + row];
              v_top = fmaxf(v_top, v_factor[i][r]);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float x = s[i][j][2 * r + c] * q_scale[j][c] * f;
                if (p.softcap > 0.f) x = p.softcap * kLog2e * tanhf(x / p.softcap);
                x = seen ? x : -INFINITY;
                s[i][j][2 * r + c] = x;
                top[j][c] = fmaxf(top[j][c], x);
              }
            }
          }
        }
        bool grown = false;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top[j][c] = fmaxf(top[j][c], __shfl_xor_sync(0xffffffffu, top[j][c], d));
            if (MODE != MODE_BF16) top[j][c] -= kF16Shift;
            grown |= top[j][c] > m[j][c];
          }
        }
        float v_unit = 1.f;
        if constexpr (MODE == MODE_E4M3) {
          // Probabilities times value factors are rounded to fp16 relative to the largest factor so far, rounded up to
          // a power of two (cv); O is in units of cv.
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) v_top = fmaxf(v_top, __shfl_xor_sync(0xffffffffu, v_top, d));
          grown |= v_top > cv;
        }
        if (__any_sync(0xffffffffu, grown)) {
          float cv_ratio = 1.f;
          if constexpr (MODE == MODE_E4M3) {
            if (v_top > cv) {
              const uint32_t e = min((__float_as_uint(v_top) >> 23) + 1, 250u);
              const float now = __uint_as_float(e << 23);
              cv_ratio = cv / now;
              cv = now;
            }
          }
#pragma unroll
          for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float now = fmaxf(m[j][c], top[j][c]);
              const float ratio = now == -INFINITY ? 1.f : exp2_fast(m[j][c] - now);
              m[j][c] = now;
              l[j][c] *= ratio;
#pragma unroll
              for (int d = 0; d < DK; ++d) {
                o[d][j][c] *= ratio * cv_ratio;
                o[d][j][2 + c] *= ratio * cv_ratio;
              }
            }
          }
        }
        if constexpr (MODE == MODE_E4M3) v_unit = 1.f / cv;
        // P^T
        uint32_t pf[MT][NT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float x[2];
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const float base = m[j][c] == -INFINITY ? 0.f : m[j][c];
                x[c] = exp2_fast(s[i][j][2 * r + c] - base);
                l[j][c] += x[c];
                if constexpr (MODE == MODE_E4M3) x[c] *= v_factor[i][r] * v_unit;
              }
              pf[i][j][r] = transpose8x8(pack2<kBf16>(x[0], x[1]));
            }
          }
        }
        // O^T
        if constexpr (MODE != MODE_E4M3) {
#pragma unroll
          for (int d = 0; d < DK; ++d) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              uint32_t a[4];
              ldmatrix4_trans(a, smem_addr(v_s) + i * 16 * S::kPitchV + v_lane + d * 32);
#pragma unroll
              for (int j = 0; j < NT; ++j) mma<kBf16>(o[d][j], a, pf[i][j][0], pf[i][j][1]);
            }
          }
        } else {
          // Lane (g, t) reads neighbouring elements of value rows 2t, 2t + 1, 2t + 8, 2t + 9; byte pairs of two rows become
          // the fragment's registers. Element e of the lane's D / 8 is row g (e even) or g + 8 (e odd) of block e / 2.
          constexpr int kWords = D / 32;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            uint32_t w[4][kWords];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const char *row = v_s + (16 * i + 2 * t + r % 2 + r / 2 * 8) * S::kPitchV;
              if constexpr (D == 64) {
                *reinterpret_cast<uint2 *>(w[r]) = *reinterpret_cast<const uint2 *>(row + 8 * g);
              } else if constexpr (D == 96) {
#pragma unroll
                for (int x = 0; x < kWords; ++x) w[r][x] = *reinterpret_cast<const uint32_t *>(row + 12 * g + 4 * x);
              } else {
#pragma unroll
                for (int x = 0; x < kWords / 4; ++x) {
                  const uint4 u = *reinterpret_cast<const uint4 *>(row + 128 * x + 16 * g);
                  w[r][4 * x] = u.x, w[r][4 * x + 1] = u.y, w[r][4 * x + 2] = u.z, w[r][4 * x + 3] = u.w;
                }
              }
            }
#pragma unroll
            for (int x = 0; x < kWords; ++x) {
              const uint32_t u0 = __byte_perm(w[0][x], w[1][x], 0x5140), u1 = __byte_perm(w[0][x], w[1][x], 0x7362);
              const uint32_t u2 = __byte_perm(w[2][x], w[3][x], 0x5140), u3 = __byte_perm(w[2][x], w[3][x], 0x7362);
              const uint32_t a0[4] = {e4m3_lo(u0), e4m3_hi(u0), e4m3_lo(u2), e4m3_hi(u2)};
              const uint32_t a1[4] = {e4m3_lo(u1), e4m3_hi(u1), e4m3_lo(u3), e4m3_hi(u3)};
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                mma<false>(o[2 * x][j], a0, pf[i][j][0], pf[i][j][1]);
                mma<false>(o[2 * x + 1][j], a1, pf[i][j][0], pf[i][j][1]);
              }
            }
          }
        }
      }
      stage = stage + 1 == S::kStages ? 0 : stage + 1;
      __syncwarp();  // all lanes are done with this stage before the next round refills it
      const int tile = cur.tile + 1;
      ends = tile == cur.n;
      advance(cur, p, S::kTileKeys);
      if (ends || cur.left <= 0) break;
    }

    // ---- the pair's (or piece's) result of this block: the warps' results joined ----
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[j][c] += __shfl_xor_sync(0xffffffffu, l[j][c], d);
        if (g == 0) {
          stats[warp * S::kHeads + 8 * j + 2 * t + c] = m[j][c];
          stats[(kWarps + warp) * S::kHeads + 8 * j + 2 * t + c] = l[j][c];
        }
      }
    }
    __syncthreads();
    float factor[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = 8 * j + 2 * t + c;
        float top = stats[col], sum = 0.f;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, stats[w * S::kHeads + col]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          sum = fmaf(exp2_fast(stats[w * S::kHeads + col] - base), stats[(kWarps + w) * S::kHeads + col], sum);
        }
        factor[j][c] = exp2_fast(m[j][c] - base) * (MODE == MODE_E4M3 ? cv : 1.f);
        if (warp == 0 && g == 0) {
          // For the writers below, in the place of warp-wise values that nobody else reads.
          stats[2 * kWarps * S::kHeads + col] = top;
          stats[(2 * kWarps + 1) * S::kHeads + col] = sum;
        }
      }
    }
    const bool whole = begins && ends;
    float *part = p.partial + (static_cast<long long>(blockIdx.x) * 2 + (begins ? 1 : 0)) * S::kHeads * (D + 2);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      // Rows [half * D / 2, + D / 2) of O^T in the order of the fragments, as [warp][head][D / 2].
#pragma unroll
      for (int dd = 0; dd < DK / 2; ++dd) {
        const int d = half * (DK / 2) + dd;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            // 16-bit: rows 16 dd + g and + 8. e4m3: the lane's elements 2 dd and 2 dd + 1.
            const int col = 8 * j + 2 * t + c % 2;
            const int row = 16 * dd + 8 * (c / 2) + g;
            merge[(warp * S::kHeads + col) * (D / 2) + row] = o[d][j][c] * factor[j][c % 2];
          }
        }
      }
      __syncthreads();
      for (int i = tid; i < n_heads * (D / 2); i += kPagedThreads) {
        const int col = i / (D / 2), at = i % (D / 2);
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) x += merge[(w * S::kHeads + col) * (D / 2) + at];
        int e;  // which element of the head this row of O^T is
        if constexpr (MODE != MODE_E4M3) {
          e = half * (D / 2) + at;
        } else {
          const int of_lane = 2 * (half * (DK / 2) + at / 16) + at % 16 / 8, group = at % 8;
          e = D <= 128 ? group * (D / 8) + of_lane : of_lane / 16 * 128 + group * 16 + of_lane % 16;
        }
        if (whole) {
          const float sum = stats[(2 * kWarps + 1) * S::kHeads + col];
          x = stats[2 * kWarps * S::kHeads + col] == -INFINITY && sum == 0.f ? 0.f : x / sum;
          const long long to = (static_cast<long long>(b) * p.heads + h0 + col) * D + e;
          if (p.out_f32) static_cast<float *>(p.out)[to] = x;
          else if (p.q_bf16) store1(static_cast<__nv_bfloat16 *>(p.out) + to, x);
          else store1(static_cast<__half *>(p.out) + to, x);
        } else {
          part[col * (D + 2) + e] = x;
        }
      }
      __syncthreads();
    }
    if (tid < n_heads) {
      const float top = stats[2 * kWarps * S::kHeads + tid], sum = stats[(2 * kWarps + 1) * S::kHeads + tid];
      if (!whole) {
        part[tid * (D + 2) + D] = top;
        part[tid * (D + 2) + D + 1] = sum;
      } else if (p.lse != nullptr) {
        p.lse[static_cast<long long>(b) * p.heads + h0 + tid] =
            top == -INFINITY && sum == 0.f ? -INFINITY : top * kLn2 + logf(sum);
      }
    }
    __syncthreads();
  }
  copies_wait<0>();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Adds the partial results of the pairs that several blocks share, in the order of the blocks. A block has one head of one
// pair; its groups of D / 2 threads take the pieces in turn, two elements a thread.
template <int D, int HEADS>
__global__ void __launch_bounds__(256) paged_join_kernel(const Params p, int tile_keys) {
  constexpr int kLanes = D / 2, kGroups = 256 / kLanes;
  __shared__ float2 sums[kGroups][kLanes];
  __shared__ float tops[kGroups], totals[kGroups];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int units = p.kv_heads * p.chunks;
  const int col = blockIdx.x % HEADS, unit = blockIdx.x / HEADS % units, b = blockIdx.x / (HEADS * units);
  const int kv = unit / p.chunks, head = kv * p.group + unit % p.chunks * HEADS + col;
  if (head >= (kv + 1) * p.group) return;
  const int n = tiles_of(visible(p.lengths[b], p.capacity, p.window), tile_keys);
  if (n == 0) return;
  const long long per = p.bases[p.batch + 1], begin = p.bases[b] + static_cast<long long>(unit) * n;
  const Owners own = owners(begin, n, per);
  if (own.first == own.last) return;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  float2 acc = make_float2(0.f, 0.f);
  float top = -INFINITY, total = 0.f;
  if (group < kGroups) {
    for (long long c = own.first + group; c <= own.last; c += kGroups) {
      const float *part = p.partial + ((c * 2 + place(own, c)) * HEADS + col) * (D + 2);
      const float2 x = *reinterpret_cast<const float2 *>(part + 2 * lane);
      const float m = part[D], s = part[D + 1];
      const float now = fmaxf(top, m), base = now == -INFINITY ? 0.f : now;
      const float keep = exp2_fast(top - base), add = exp2_fast(m - base);
      acc.x = fmaf(x.x, add, acc.x * keep);
      acc.y = fmaf(x.y, add, acc.y * keep);
      total = fmaf(s, add, total * keep);
      top = now;
    }
    sums[group][lane] = acc;
    if (lane == 0) tops[group] = top, totals[group] = total;
  }
  __syncthreads();
  if (threadIdx.x >= kLanes) return;
  float all = tops[0];
#pragma unroll
  for (int i = 1; i < kGroups; ++i) all = fmaxf(all, tops[i]);
  const float base = all == -INFINITY ? 0.f : all;
  acc = make_float2(0.f, 0.f);
  total = 0.f;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const float f = exp2_fast(tops[i] - base);
    acc.x = fmaf(sums[i][lane].x, f, acc.x);
    acc.y = fmaf(sums[i][lane].y, f, acc.y);
    total = fmaf(totals[i], f, total);
  }
  const bool none = all == -INFINITY && total == 0.f;
  const float inv = none ? 0.f : 1.f / total;
  const long long to = (static_cast<long long>(b) * p.heads + head) * D + 2 * lane;
  if (p.out_f32) {
    *reinterpret_cast<float2 *>(static_cast<float *>(p.out) + to) = make_float2(acc.x * inv, acc.y * inv);
  } else {
    const uint32_t w = p.q_bf16 ? pack2<true>(acc.x * inv, acc.y * inv) : pack2<false>(acc.x * inv, acc.y * inv);
    *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(p.out) + to) = w;
  }
  if (lane == 0 && p.lse != nullptr) {
    p.lse[static_cast<long long>(b) * p.heads + head] = none ? -INFINITY : all * kLn2 + logf(total);
  }
}

// ---- host side ----------------------------------------------------------------------------------------------------

constexpr int kMostBlocksPerSm = 2;
// Tiles that a block takes at least: below that its fixed costs weigh more than the loads that another SM would take over.
constexpr int kLeastTiles = 2;

int heads_per_unit(int group, int dim) { return group > 8 && dim <= 128 ? 16 : 8; }

template <int D, int NT, int MODE>
int launch(Params p, cudaStream_t s) {
  using S = Shape<D, NT, MODE>;
  p.blocks = device_sm_count() * S::kBlocks;
  auto kernel = paged_kernel<D, NT, MODE>;
  // The attribute belongs to the device's context: set once for each device.
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  kernel<<<p.blocks, kPagedThreads, S::kSmem, s>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (p.capacity <= S::kTileKeys) return 0;  // no pair has two tiles: nothing to join
  // The join's blocks may start while the last blocks above are running; they wait for them before they read.
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.batch) * p.kv_heads * p.chunks * S::kHeads);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<D, S::kHeads>, p, static_cast<int>(S::kTileKeys));
}

template <int D, int MODE>
int launch_heads(const Params &p, cudaStream_t s) {
  if constexpr (D <= 128) {
    if (heads_per_unit(p.group, D) == 16) return launch<D, 2, MODE>(p, s);
  }
  return launch<D, 1, MODE>(p, s);
}

template <int D>
int launch_mode(const Params &p, int cache_type, cudaStream_t s) {
  switch (cache_type) {
    case ATTN_BF16: return launch_heads<D, MODE_BF16>(p, s);
    case ATTN_F16: return launch_heads<D, MODE_F16>(p, s);
    case ATTN_E4M3: return launch_heads<D, MODE_E4M3>(p, s);
    default: return cudaErrorInvalidValue;
  }
}

bool refuse_sizes(const KvCacheArgs &c, int batch, int heads) {
  return (c.dim != 64 && c.dim != 96 && c.dim != 128 && c.dim != 256) || batch < 0 || heads < 1 || c.kv_heads < 1 ||
         heads % c.kv_heads || c.pages < 0 || c.page_shift < 0 || c.page_shift > 20 ||
         (static_cast<long long>(c.pages) * c.kv_heads << c.page_shift) > 0x7fffffffll ||
         static_cast<long long>(batch) * c.kv_heads * ((heads / c.kv_heads + 7) / 8) * 16 > 0x7fffffffll;
}

size_t partial_floats(const KvCacheArgs &c, int heads, int blocks) {
  return static_cast<size_t>(blocks) * 2 * heads_per_unit(heads / c.kv_heads, c.dim) * (c.dim + 2);
}

}  // namespace
}  // namespace attn

using namespace attn;

size_t paged_attention_workspace(const KvCacheArgs &c, int batch, int heads) {
  if (refuse_sizes(c, batch, heads)) return 0;
  return (static_cast<size_t>(batch) + 2) * 8 + partial_floats(c, heads, device_sm_count() * kMostBlocksPerSm) * 4;
}

int paged_attention(const KvCacheArgs &c, const PagedAttentionArgs &a, void *workspace, size_t workspace_bytes,
                    void *stream) {
  if (refuse_sizes(c, a.batch, a.heads) || (c.type == ATTN_E4M3 && (!c.k_scale || !c.v_scale)) ||
      (a.q_type != ATTN_BF16 && a.q_type != ATTN_F16) || (c.type != ATTN_E4M3 && c.type != a.q_type) ||
      (a.out_type != a.q_type && a.out_type != ATTN_F32) || a.window < 0 || a.max_pages < 0 ||
      (static_cast<long long>(a.max_pages) << c.page_shift) > 0x7fffffffll - 256 ||
      workspace_bytes < paged_attention_workspace(c, a.batch, a.heads)) {
    return cudaErrorInvalidValue;
  }
  if (a.batch == 0) return 0;
  Params p{};
  p.q = a.q;
  p.q_token = a.q_token;
  p.q_head = a.q_head;
  p.k = static_cast<const char *>(c.k);
  p.v = static_cast<const char *>(c.v);
  p.k_scale = c.k_scale;
  p.v_scale = c.v_scale;
  p.table = a.block_table;
  p.table_stride = a.table_stride;
  p.lengths = a.lengths;
  p.batch = a.batch;
  p.heads = a.heads;
  p.kv_heads = c.kv_heads;
  p.group = a.heads / c.kv_heads;
  p.chunks = (p.group + heads_per_unit(p.group, c.dim) - 1) / heads_per_unit(p.group, c.dim);
  p.pages = c.pages;
  p.shift = c.page_shift;
  p.capacity = a.max_pages << c.page_shift;
  p.window = a.window;
  p.scale = a.scale;
  p.softcap = a.softcap;
  p.out = a.out;
  p.lse = a.lse;
  p.q_bf16 = a.q_type == ATTN_BF16;
  p.out_f32 = a.out_type == ATTN_F32;
  p.bases = static_cast<long long *>(workspace);
  p.partial = reinterpret_cast<float *>(p.bases + a.batch + 2);
  p.least = kLeastTiles;
  // A block counts its tiles in 32 bits (tiles have at least 64 keys).
  if (static_cast<long long>(a.batch) * c.kv_heads * p.chunks > 0x7fffffffll * device_sm_count() / (p.capacity / 64 + 1)) {
    return cudaErrorInvalidValue;
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (c.dim) {
    case 64: return launch_mode<64>(p, c.type, s);
    case 96: return launch_mode<96>(p, c.type, s);
    case 128: return launch_mode<128>(p, c.type, s);
    default: return launch_mode<256>(p, c.type, s);
  }
}

}  // namespace kernels
}  // namespace rocshmem
