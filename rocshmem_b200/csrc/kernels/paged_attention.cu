// Attention of one new token per sequence over a paged cache, split over the cache's length and joined.
//
//   s_j = scale q.k_j  (capped: c tanh(s_j / c))
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   lse = m + log sum_j exp(s_j - m)
//
// A key and a value are read once and used by the 1 - 16 query heads that share them, so memory bounds the kernel:
// about 23 bytes a cycle and SM have to arrive, and the arithmetic only has to keep up. The products run on warp-level
// matrix instructions with the KEYS as the tile's 16 rows and the query heads as its 8 columns: a group of up to eight
// heads wastes nothing (with the heads as rows, half and more of each instruction would be padding), and 16 keys a warp
// are enough to feed it. tcgen05 needs 128 rows to a tile and accumulators in TMEM; it has nothing to give where the
// tensor pipe idles.
//
//   S^T [16 keys, 8 heads] = K [16, D] Q^T [D, 8]          A = K rows as they lie, B = queries, kept in registers
//   O^T [D, 8 heads]      += V^T [D, 16 keys] P^T [16, 8]  A = V transposed on the way out of shared memory
//
// The accumulator layout of S^T differs from the operand layout of P^T by a transposition of 8 x 8 blocks (movmatrix).
// Both products have a head's values in the same lanes, so rescaling O by the change of the maximum needs no exchange.
//
// Blocks are single warps that work on their own. The line of all tiles (attention_plan.hpp) is dealt to them in equal
// shares; a warp streams its tiles through a ring of stages (cp.async; rows behind the end, of bad pages and before the
// window arrive as zeros and score -inf) with a running maximum and sum, and its loads run ahead from one pair into the
// next. There is no barrier. A pair that lies in several shares leaves unnormalised partial results, which
// paged_join_kernel adds in the order of the shares: results do not depend on which warp is done first.
//
// e4m3 caches: codes become fp16 exactly (cvt), a key's factor multiplies its score, a value's factor its probability.
// They are bound by instructions as much as by memory: 32 keys a step need 650 (two steps of 16 keys took 15 % longer).
//
// Measured on one B200, 128 elements a head, launches one after the other without the host: 64 sequences of 1024 - 4096
// tokens, 32 / 8 heads, bf16, 117 us for 675 MB (5.8 TB/s; a device copy: 6.4); two sequences of 130 - 520 thousand,
// 64 / 8 heads, e4m3, 312 us for 1.94 GB (6.2). Public calls in a loop: 118 us for 670 MB (5.7) and 328 us for 2.03 GB
// (6.2). The join takes 5 us of it. What is left in the first is the start, 4 us until data arrives, and the SMs that
// end last (see Shape). Farther from memory: 16 heads a key head in e4m3 (54 us for a floor of 27: the softmax's
// arithmetic at two warps a scheduler) and in bf16 with 64 elements (42 for 26), one sequence of 32768 tokens (35 for
// 21: start, join), 256 sequences of 512 tokens (72 for 54, e4m3 51 for 28: each pair begins with a wait for its
// queries).
#include "attention_common.cuh"

#include <atomic>

namespace rocshmem {
namespace kernels {

namespace attn {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Probabilities are at most 1. Where they are rounded to fp16 they are scaled by 2^14 first, so that one down to 2^-28
// of the largest keeps all its bits and none above 2^-39 is lost from a long sum; the factor is in the sum as well and
// cancels.
constexpr float kF16Shift = 14.f;

enum Mode : int { MODE_BF16 = 0, MODE_F16 = 1, MODE_E4M3 = 2 };

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
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
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
                 "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
                 "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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
template <bool BF16>
__device__ __forceinline__ void unpack2(uint32_t w, float &lo, float &hi) {
  if (BF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    lo = f.x, hi = f.y;
  }
}
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// c tanh(x / c) in base 2, with in = 1 / c and back = c log2(e). Up to one, where most scores are, tanh y is Lambert's
// continued fraction y / (1 + y^2 / (3 + y^2 / (5 + y^2 / (7 + y^2 / 9)))) as a quotient (off by 6e-8 of it at most),
// beyond 1 - 2 / (exp(2y) + 1), whose error there is one of the last bits too. tanhf cost a fifth of the kernel's time.
__device__ __forceinline__ float cap2(float x, float in, float back) {
  const float y = x * in, y2 = y * y;
  const float near = y * fmaf(y2 + 105.f, y2, 945.f) * reciprocal(fmaf(fmaf(15.f, y2, 420.f), y2, 945.f));
  const float far = fmaf(-2.f, reciprocal(exp2_fast(y * (2.f * kLog2e)) + 1.f), 1.f);
  return back * (fabsf(y) <= 1.f ? near : far);
}

// Shared memory and tile sizes of one instantiation. Rows are padded so that the accesses of a fragment fall into
// different banks: 16 bytes for 16-bit rows (ldmatrix), for e4m3 32 bytes a key row (8 bytes a lane from four rows) and
// 16 a value row (up to 16 bytes a lane from every other row). With 96 e4m3 elements a key row already has that stride.
template <int D, int NT, int MODE>
struct Shape {
  static constexpr int kElem = MODE == MODE_E4M3 ? 1 : 2;
  static constexpr int kKeys = MODE == MODE_E4M3 && D <= 128 ? 32 : 16;  // keys a warp takes a step
  static constexpr int kRowBytes = D * kElem;
  static constexpr int kPitchK = kRowBytes + (MODE == MODE_E4M3 ? (D == 96 ? 0 : 32) : 16);
  static constexpr int kPitchV = kRowBytes + 16;
  static constexpr int kScales = MODE == MODE_E4M3 ? 2 * kKeys * 4 : 0;
  // one warp's stage; its last word: which rows are seen
  static constexpr int kStage = kKeys * (kPitchK + kPitchV) + kScales + 16;
  static constexpr int kHeads = 8 * NT;
  static constexpr int kFrags = D / 16 * NT;               // of O^T, four values a lane
  static constexpr int kPart = kFrags * 128 + 2 * kHeads;  // floats of a partial result: O^T, maxima (base 2), sums
  // Two stages: one tile on its way while the other is used. e4m3 is bound by instructions and takes as many warps as
  // its registers allow. 16-bit caches are bound by memory and want 64 - 70 KB on their way for each SM, no more: SMs
  // of large GPCs get less of the bandwidth than others, and the further the queues reach, the later they end (128
  // elements, 64 sequences, blocks x stages an SM: 8 x 2 119 us, 12 x 2 123, 5 x 4 123, 8 x 3 127).
  static constexpr int kStages = 2;
  static constexpr int kWarpsByRegisters = NT == 2 ? (D == 64 ? 12 : 8) : D == 64 ? 16 : D == 96 ? 12 : 8;
  static constexpr int kWarpsByBytes = 70 * 1024 / kStage;
  static constexpr int kBlocks =
      MODE == MODE_E4M3 || kWarpsByBytes > kWarpsByRegisters ? kWarpsByRegisters : kWarpsByBytes;
  static constexpr int kSmem = kStages * kStage;
  static constexpr int kTeam = 8 * kSmem <= 226 * 1024 ? 8 : 4;  // warps of a block of paged_short_kernel
  static_assert(kBlocks * (kSmem + 1024) <= 228 * 1024 && kPitchK % 16 == 0 && kPitchV % 16 == 0 && kStage % 16 == 0,
      "alignment");
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
  float *partial;     // [shares][2][kPart]
  int2 *spans;        // [batch][units]: the first and the last share that a pair lies in
  int blocks, least;
};

// Walks the tiles of a warp's share in order.
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

// Which element of its head row r (0 - 15) of block d of O^T is. e4m3: see where the value rows are read.
template <int D, int MODE>
__device__ __forceinline__ int element(int d, int r) {
  if (MODE != MODE_E4M3) return 16 * d + r;
  const int of_lane = 2 * d + r / 8, group = r % 8;
  return D <= 128 ? group * (D / 8) + of_lane : of_lane / 16 * 128 + group * 16 + of_lane % 16;
}

__device__ __forceinline__ void store_out(const Params &p, long long at, float x) {
  if (p.out_f32) static_cast<float *>(p.out)[at] = x;
  else if (p.q_bf16) store1(static_cast<__nv_bfloat16 *>(p.out) + at, x);
  else store1(static_cast<__half *>(p.out) + at, x);
}

// For the two heads of a lane's columns in group j: the factor that makes sums of p v results, and, by one lane each,
// the lse.
template <int NT>
__device__ __forceinline__ void finish(const Params &p, long long row0, int n_heads, int j, int lane,
    const float (&m)[2], const float (&l)[2], float (&inv)[2]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int col = 8 * j + 2 * (lane % 4) + c;
    const bool none = m[c] == -INFINITY && l[c] == 0.f;
    inv[c] = none ? 0.f : 1.f / l[c];
    if (lane < 4 && p.lse != nullptr && col < n_heads) p.lse[row0 + col] = none ? -INFINITY : m[c] * kLn2 + logf(l[c]);
  }
}

// Fragment (d, j) of O^T times the heads' factors, to the result. All lanes of the warp call it.
template <int D, int MODE>
__device__ __forceinline__ void store_fragment(const Params &p, long long row0, int n_heads, int j, int d, int lane,
    const float (&o)[4], const float (&inv)[2]) {
  const int g = lane / 4, t = lane % 4;
  if (p.out_f32) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int col = 8 * j + 2 * t + c % 2;
      if (col < n_heads) {
        static_cast<float *>(p.out)[(row0 + col) * D + element<D, MODE>(d, 8 * (c / 2) + g)] = o[c] * inv[c % 2];
      }
    }
  } else if constexpr (MODE == MODE_E4M3) {
    // A lane's rows g and g + 8 are neighbouring elements.
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int col = 8 * j + 2 * t + c;
      const float x = o[c] * inv[c], y = o[2 + c] * inv[c];
      if (col < n_heads) {
        *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(p.out) + (row0 + col) * D + element<D, MODE>(d, g)) =
            p.q_bf16 ? pack2<true>(x, y) : pack2<false>(x, y);
      }
    }
  } else {
    // Transposed, a lane has two neighbouring elements of head g.
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t w = transpose8x8(pack2<MODE == MODE_BF16>(o[2 * r] * inv[0], o[2 * r + 1] * inv[1]));
      if (8 * j + g < n_heads) {
        uint16_t *const to = static_cast<uint16_t *>(p.out) + (row0 + 8 * j + g) * D;
        *reinterpret_cast<uint32_t *>(to + 16 * d + 8 * r + 2 * t) = w;
      }
    }
  }
}

// Streams the tiles of a warp's share, from `cur` on. done(...) is called at the end of every pair, or of the share's
// part of one, with the accumulators of O^T (e4m3: in units of cv), maxima and sums of the lane's columns, and whether
// the pair begins and ends here.
template <int D, int NT, int MODE, typename F>
__device__ __forceinline__ void run_share(const Params &p, char *ring, Cursor cur, int lane, F done) {
  using S = Shape<D, NT, MODE>;
  constexpr bool kBf16 = MODE == MODE_BF16;
  constexpr int kKeys = S::kKeys, MT = kKeys / 16, DK = D / 16;
  const int g = lane / 4, t = lane % 4;
  Cursor ahead = cur;

  // ---- loads: `ahead` runs kStages - 1 tiles before `cur`; a tile's page is looked up a step before its rows are ----
  const uint32_t stages = smem_addr(ring);
  struct Next {
    int page, pos, head;  // of the lane's key; pos < 0: none
  };
  auto look_up = [&](const Cursor &c) -> Next {
    const int pos = c.first + c.tile * kKeys + lane;
    if (c.left <= 0 || (kKeys < 32 && lane >= kKeys) || pos >= c.end) return Next{0, -1, 0};
    return Next{p.table[c.b * p.table_stride + (pos >> p.shift)], pos, c.unit / p.chunks};
  };
  // A row is kChunks pieces of 16 bytes. Where whole rows make up a warp's copy, a lane has the same piece of every
  // kEach-th row, and all its addresses are one register and constants.
  constexpr unsigned kChunks = S::kRowBytes / 16, kCopies = kKeys * kChunks / 32;
  static_assert(kKeys * kChunks % 32 == 0, "whole warps");
  constexpr bool kEven = 32 % kChunks == 0;
  constexpr unsigned kEach = kEven ? 32 / kChunks : 1;
  const unsigned my_row = kEven ? lane / kChunks : 0, my_piece = kEven ? lane % kChunks : 0;
  const char *const my_k = p.k + my_piece * 16, *const my_v = p.v + my_piece * 16;
  const uint32_t my_to = stages + my_row * S::kPitchK + my_piece * 16;
  const uint32_t my_to_v = stages + kKeys * S::kPitchK + my_row * S::kPitchV + my_piece * 16;
  auto load = [&](int stage, const Next &key) {
    const int row = key.pos < 0 ? -1 : page_row(key.page, p.pages, key.pos, p.shift, p.kv_heads, key.head);
    const uint32_t mask = __ballot_sync(0xffffffffu, row >= 0);
    const uint32_t at_stage = stage * S::kStage;
    if (lane == 0) *reinterpret_cast<uint32_t *>(ring + at_stage + S::kStage - 16) = mask;
#pragma unroll
    for (unsigned i = 0; i < kCopies; ++i) {
      const unsigned at = i * 32 + lane;
      const unsigned r = kEven ? i * kEach + my_row : at / kChunks, c = kEven ? 0 : at % kChunks;
      const int from = __shfl_sync(0xffffffffu, row, r);
      const uint32_t bytes = from < 0 ? 0 : 16;
      const unsigned at_row = static_cast<unsigned>(max(from, 0));
      const unsigned long long off = static_cast<unsigned long long>(at_row) * S::kRowBytes;
      const uint32_t to_k = kEven ? i * kEach * S::kPitchK : r * S::kPitchK + c * 16;
      const uint32_t to_v = kEven ? i * kEach * S::kPitchV : r * S::kPitchV + c * 16;
      copy16(my_to + at_stage + to_k, my_k + off + c * 16, bytes);
      copy16(my_to_v + at_stage + to_v, my_v + off + c * 16, bytes);
    }
    if constexpr (MODE == MODE_E4M3) {
      const uint32_t to = stages + at_stage + kKeys * (S::kPitchK + S::kPitchV) + 4 * lane;
      if constexpr (kKeys == 32) {
        copy4(to, p.k_scale + max(row, 0), row < 0 ? 0 : 4);
        copy4(to + 4 * kKeys, p.v_scale + max(row, 0), row < 0 ? 0 : 4);
      } else {
        const int from = __shfl_sync(0xffffffffu, row, lane % 16);
        copy4(to, (lane < 16 ? p.k_scale : p.v_scale) + max(from, 0), from < 0 ? 0 : 4);
      }
    }
  };
  Next next = look_up(ahead);
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) {
    if (ahead.left > 0) {
      load(i, next);
      advance(ahead, p, kKeys);
      next = look_up(ahead);
    }
    copies_commit();
  }
  int stage = 0, load_stage = S::kStages - 1;

  // ---- pairs ----
  const float cap_in = 1.f / p.softcap, cap_back = p.softcap * kLog2e;
  // ldmatrix: 16 keys x 16 elements
  const int k_lane = (lane % 16) * S::kPitchK + (lane / 16) * 16;
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
        // A head's largest magnitude brought to [1, 2) by a power of two. bf16 values (8 bits) then fit fp16 exactly
        // down to 2^-17, fp16 values (11 bits) down to 2^-14; what is smaller is rounded to steps of 2^-24, off by
        // 2^-25 at most, half of what fp32 would round off the largest element's product.
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
    const Cursor pair = cur;
    bool ends = false;
    while (true) {
      copies_wait<S::kStages - 2>();
      __syncwarp();
      if (ahead.left > 0) {
        load(load_stage, next);
        advance(ahead, p, kKeys);
        next = look_up(ahead);
      }
      copies_commit();
      load_stage = load_stage + 1 == S::kStages ? 0 : load_stage + 1;

      const char *k_s = ring + stage * S::kStage, *v_s = k_s + kKeys * S::kPitchK;
      const uint32_t k_a = stages + stage * S::kStage + k_lane;
      const uint32_t v_a = stages + stage * S::kStage + kKeys * S::kPitchK + v_lane;
      const float *f_s = reinterpret_cast<const float *>(v_s + kKeys * S::kPitchV);
      const uint32_t mask = *reinterpret_cast<const uint32_t *>(k_s + S::kStage - 16);
      {
        // S^T
        float s[MT][NT][4] = {};
        if constexpr (MODE != MODE_E4M3) {
#pragma unroll
          for (int kk = 0; kk < DK; ++kk) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              uint32_t a[4];
              ldmatrix4(a, k_a + i * 16 * S::kPitchK + kk * 32);
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
              uint32_t a0[4], a1[4];
              e4m3_pairs(lo.x, a0[0], a0[2]);
              e4m3_pairs(hi.x, a0[1], a0[3]);
              e4m3_pairs(lo.y, a1[0], a1[2]);
              e4m3_pairs(hi.y, a1[1], a1[3]);
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
              v_top = fmaxf(v_top, fabsf(v_factor[i][r]));
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float x = s[i][j][2 * r + c] * (q_scale[j][c] * f);
                if (p.softcap > 0.f) x = cap2(x, cap_in, cap_back);
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
        // P^T, as a value rounded to the operand's type and the rounded rest: of one part alone the rounding of
        // bf16 (2^-8) or fp16 (2^-11) would be as large as that of the result. Two are off by 2^-17 and 2^-23. The
        // second costs nothing where memory bounds (64 sequences of 1024 - 4096 tokens in bf16: 117 us both), 8 % with
        // 16 heads a key head in e4m3 (54.0 us against 49.7).
        uint32_t pf[MT][NT][2], pr[MT][NT][2];
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
              const uint32_t top2 = pack2<kBf16>(x[0], x[1]);
              pf[i][j][r] = transpose8x8(top2);
              float y[2];
              unpack2<kBf16>(top2, y[0], y[1]);
              pr[i][j][r] = transpose8x8(pack2<kBf16>(x[0] - y[0], x[1] - y[1]));
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
              ldmatrix4_trans(a, v_a + i * 16 * S::kPitchV + d * 32);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                mma<kBf16>(o[d][j], a, pf[i][j][0], pf[i][j][1]);
                mma<kBf16>(o[d][j], a, pr[i][j][0], pr[i][j][1]);
              }
            }
          }
        } else {
          // Lane (g, t) reads neighbouring elements of value rows 2t, 2t + 1, 2t + 8, 2t + 9; byte pairs of two rows
          // become the fragment's registers. Element e of the lane's D / 8 is row g (e even) or g + 8 (e odd) of block
          // e / 2.
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
              uint32_t a0[4], a1[4];
              e4m3_pairs(u0, a0[0], a0[1]);
              e4m3_pairs(u2, a0[2], a0[3]);
              e4m3_pairs(u1, a1[0], a1[1]);
              e4m3_pairs(u3, a1[2], a1[3]);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                mma<false>(o[2 * x][j], a0, pf[i][j][0], pf[i][j][1]);
                mma<false>(o[2 * x + 1][j], a1, pf[i][j][0], pf[i][j][1]);
                mma<false>(o[2 * x][j], a0, pr[i][j][0], pr[i][j][1]);
                mma<false>(o[2 * x + 1][j], a1, pr[i][j][0], pr[i][j][1]);
              }
            }
          }
        }
      }
      stage = stage + 1 == S::kStages ? 0 : stage + 1;
      __syncwarp();  // all lanes are done with this stage before the next round refills it
      const int tile = cur.tile + 1;
      ends = tile == cur.n;
      advance(cur, p, kKeys);
      if (ends || cur.left <= 0) break;
    }

#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[j][c] += __shfl_xor_sync(0xffffffffu, l[j][c], d);
      }
    }
    done(pair, begins, ends, h0, n_heads, o, m, l, cv);
  }
  copies_wait<0>();
}

// A partial result: fragments as they lie in the lanes, then maxima and sums of the columns.
template <int D, int NT, int MODE>
__device__ __forceinline__ void store_part(float *part, int lane, const float (&o)[D / 16][NT][4],
    const float (&m)[NT][2], const float (&l)[NT][2], float cv) {
  using S = Shape<D, NT, MODE>;
  const float f = MODE == MODE_E4M3 ? cv : 1.f;
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      reinterpret_cast<float4 *>(part)[(d * NT + j) * 32 + lane] =
          make_float4(o[d][j][0] * f, o[d][j][1] * f, o[d][j][2] * f, o[d][j][3] * f);
    }
  }
  if (lane < 4) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      *reinterpret_cast<float2 *>(part + S::kFrags * 128 + 8 * j + 2 * lane) = make_float2(m[j][0], m[j][1]);
      *reinterpret_cast<float2 *>(part + S::kFrags * 128 + S::kHeads + 8 * j + 2 * lane) =
          make_float2(l[j][0], l[j][1]);
    }
  }
}

// What a thread of a join has: the four values that a lane had of one fragment, and its two columns' maxima and sums.
struct Joined {
  float4 o;
  float2 m, l;
};
__device__ __forceinline__ Joined nothing() {
  return Joined{make_float4(0.f, 0.f, 0.f, 0.f), make_float2(-INFINITY, -INFINITY), make_float2(0.f, 0.f)};
}
__device__ __forceinline__ void add(Joined &a, const Joined &x) {
  const float2 now = make_float2(fmaxf(a.m.x, x.m.x), fmaxf(a.m.y, x.m.y));
  const float bx = now.x == -INFINITY ? 0.f : now.x, by = now.y == -INFINITY ? 0.f : now.y;
  const float kx = exp2_fast(a.m.x - bx), ky = exp2_fast(a.m.y - by);
  const float ax = exp2_fast(x.m.x - bx), ay = exp2_fast(x.m.y - by);
  a.o.x = fmaf(x.o.x, ax, a.o.x * kx);
  a.o.y = fmaf(x.o.y, ay, a.o.y * ky);
  a.o.z = fmaf(x.o.z, ax, a.o.z * kx);
  a.o.w = fmaf(x.o.w, ay, a.o.w * ky);
  a.l.x = fmaf(x.l.x, ax, a.l.x * kx);
  a.l.y = fmaf(x.l.y, ay, a.l.y * ky);
  a.m = now;
}
template <int D, int NT, int MODE>
__device__ __forceinline__ Joined load_part(const float *part, int at) {
  using S = Shape<D, NT, MODE>;
  const int col = 8 * (at / 32 % NT) + 2 * (at % 4);
  return Joined{reinterpret_cast<const float4 *>(part)[at],
      *reinterpret_cast<const float2 *>(part + S::kFrags * 128 + col),
                *reinterpret_cast<const float2 *>(part + S::kFrags * 128 + S::kHeads + col)};
}
// The result of fragment at / 32. All lanes of the warp call it.
template <int D, int NT, int MODE>
__device__ __forceinline__ void store_joined(const Params &p, int b, int unit, int at, const Joined &a) {
  using S = Shape<D, NT, MODE>;
  const int lane = at % 32, d = at / 32 / NT, j = at / 32 % NT;
  const int kv = unit / p.chunks, h0 = kv * p.group + unit % p.chunks * S::kHeads;
  const int n_heads = min(S::kHeads, (kv + 1) * p.group - h0);
  const float v[4] = {a.o.x, a.o.y, a.o.z, a.o.w}, tops[2] = {a.m.x, a.m.y}, sums[2] = {a.l.x, a.l.y};
  float inv[2];
  // One warp for each group of heads writes the lse.
  finish<NT>(p, static_cast<long long>(b) * p.heads + h0, d == 0 ? n_heads : 0, j, lane, tops, sums, inv);
  store_fragment<D, MODE>(p, static_cast<long long>(b) * p.heads + h0, n_heads, j, d, lane, v, inv);
}

template <int D, int NT, int MODE>
__global__ void __launch_bounds__(32, Shape<D, NT, MODE>::kBlocks) paged_kernel(const Params p) {
  using S = Shape<D, NT, MODE>;
  constexpr int kKeys = S::kKeys, DK = D / 16;
  extern __shared__ __align__(16) char ring[];
  const int lane = threadIdx.x;
  const int units = p.kv_heads * p.chunks;

  // ---- the line of tiles ----
  // Lanes take neighbouring sequences, `per_lane` each; a scan over the lanes gives each one its first tile.
  const int per_lane = (p.batch + 31) / 32, b_lo = min(lane * per_lane, p.batch), b_hi = min(b_lo + per_lane, p.batch);
  auto tiles_at = [&](int b) {
    return static_cast<long long>(tiles_of(visible(p.lengths[b], p.capacity, p.window), kKeys)) * units;
  };
  long long mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += tiles_at(b);
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  const long long total = __shfl_sync(0xffffffffu, upto, 31), per = per_share(total, p.blocks, p.least);
  // The join may be set up from here on; it waits for the end of this grid before it reads.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // The lane whose sequences hold the share's first tile finds the sequence.
  const long long t0 = per * blockIdx.x, t1 = min(total, t0 + per);
  const bool holds = t0 < t1 && t0 >= upto - mine && t0 < upto;
  int first_b = b_lo;
  long long into = t0 - (upto - mine);
  if (holds) {
    for (long long n = tiles_at(first_b); into >= n; n = tiles_at(first_b)) {
      into -= n;
      ++first_b;
    }
  }
  // A sequence that sees nothing gets its result here.
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    const Span s = visible(p.lengths[b], p.capacity, p.window);
    if (s.end > s.first) continue;
    for (int i = lane; i < p.heads * D; i += 32) store_out(p, static_cast<long long>(b) * p.heads * D + i, 0.f);
    for (int i = lane; i < units; i += 32) p.spans[static_cast<long long>(b) * units + i] = make_int2(0, 0);
    if (p.lse != nullptr) {
      for (int i = lane; i < p.heads; i += 32) p.lse[static_cast<long long>(b) * p.heads + i] = -INFINITY;
    }
  }
  if (t0 >= t1) return;
  const int from = __ffs(__ballot_sync(0xffffffffu, holds)) - 1;
  Cursor cur;
  cur.b = __shfl_sync(0xffffffffu, first_b, from);
  into = __shfl_sync(0xffffffffu, into, from);
  enter(cur, p, kKeys);
  cur.unit = static_cast<int>(into / cur.n);
  cur.tile = static_cast<int>(into - static_cast<long long>(cur.unit) * cur.n);
  cur.left = static_cast<int>(t1 - t0);
  run_share<D, NT, MODE>(p, ring, cur, lane, [&](const Cursor &pair, bool begins, bool ends, int h0, int n_heads,
      float (&o)[DK][NT][4], float (&m)[NT][2], float (&l)[NT][2], float cv) {
    if (begins && lane == 0) {
      const int share = blockIdx.x;
      p.spans[static_cast<long long>(pair.b) * units + pair.unit] =
          make_int2(share, last_share(share, pair.n, pair.left, static_cast<int>(per)));
    }
    if (!(begins && ends)) {
      store_part<D, NT, MODE>(p.partial + (static_cast<long long>(blockIdx.x) * 2 + (begins ? 1 : 0)) * S::kPart,
          lane, o, m, l, cv);
      return;
    }
    const long long row0 = static_cast<long long>(pair.b) * p.heads + h0;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float inv[2];
      finish<NT>(p, row0, n_heads, j, lane, m[j], l[j], inv);
      if constexpr (MODE == MODE_E4M3) inv[0] *= cv, inv[1] *= cv;
#pragma unroll
      for (int d = 0; d < DK; ++d) store_fragment<D, MODE>(p, row0, n_heads, j, d, lane, o[d][j], inv);
    }
  });
}

// Short caches: a block has one pair, its warps take equal parts of the pair's tiles and join their results through the
// ring's memory. One launch instead of two, for calls that are bound by latency.
template <int D, int NT, int MODE>
__global__ void __launch_bounds__(32 * Shape<D, NT, MODE>::kTeam) paged_short_kernel(const Params p) {
  using S = Shape<D, NT, MODE>;
  constexpr int DK = D / 16, kTeam = S::kTeam;
  extern __shared__ __align__(16) char rings[];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, units = p.kv_heads * p.chunks;
  char *const ring = rings + warp * S::kSmem;
  Cursor cur{};
  cur.b = blockIdx.x / units;
  cur.unit = blockIdx.x % units;
  enter(cur, p, S::kKeys);
  cur.tile = cur.n * warp / kTeam;
  cur.left = cur.n * (warp + 1) / kTeam - cur.tile;
  float *const part = reinterpret_cast<float *>(ring);
  static_assert(S::kPart * 4 <= S::kSmem, "a part fits the ring");
  if (cur.left > 0) {
    run_share<D, NT, MODE>(p, ring, cur, lane, [&](const Cursor &, bool, bool, int, int, float (&o)[DK][NT][4],
        float (&m)[NT][2], float (&l)[NT][2], float cv) {
      copies_wait<0>();
      __syncwarp();
      store_part<D, NT, MODE>(part, lane, o, m, l, cv);
    });
  }
  __syncthreads();
  for (int at = threadIdx.x; at < S::kFrags * 32; at += 32 * kTeam) {
    Joined a = nothing();
#pragma unroll
    for (int w = 0; w < kTeam; ++w) {
      if (cur.n * (w + 1) / kTeam > cur.n * w / kTeam) {
        add(a, load_part<D, NT, MODE>(reinterpret_cast<const float *>(rings + w * S::kSmem), at));
      }
    }
    store_joined<D, NT, MODE>(p, cur.b, cur.unit, at, a);
  }
}

// Adds the partial results of the pairs that several warps share, in the order of the shares. A thread has the four
// values that a lane had of one fragment; a block GROUPS sets of such threads, which take the parts in turn.
template <int D, int NT, int MODE, int GROUPS>
__global__ void __launch_bounds__(256) paged_join_kernel(const Params p) {
  using S = Shape<D, NT, MODE>;
  constexpr int kLanes = 256 / GROUPS, kAhead = 4;
  __shared__ Joined shared[GROUPS > 1 ? GROUPS : 1][GROUPS > 1 ? kLanes : 1];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int2 own = p.spans[blockIdx.x];
  if (own.x == own.y) return;
  const int group = threadIdx.x / kLanes, at = blockIdx.y * kLanes + threadIdx.x % kLanes;
  const bool has = at < S::kFrags * 32;
  Joined a = nothing();
  if (has) {
    for (int c0 = own.x + group; c0 <= own.y; c0 += kAhead * GROUPS) {
      Joined x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int c = c0 + i * GROUPS;
        if (c > own.y) break;
        x[i] = load_part<D, NT, MODE>(p.partial + (static_cast<long long>(c) * 2 + place(own.x, c)) * S::kPart, at);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (c0 + i * GROUPS > own.y) break;
        add(a, x[i]);
      }
    }
  }
  if constexpr (GROUPS > 1) {
    const int at_s = threadIdx.x % kLanes;
    shared[group][at_s] = a;
    __syncthreads();
    if (group != 0) return;
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) add(a, shared[i][at_s]);
  }
  const int units = p.kv_heads * p.chunks;
  if (has) store_joined<D, NT, MODE>(p, blockIdx.x / units, blockIdx.x % units, at, a);
}

// ---- host side ----------------------------------------------------------------------------------------------------

// Keys a warp of paged_short_kernel, at most: with more, splitting over more SMs pays for a second launch. 128
// elements, bf16, 32 pairs, one launch against two: 128 keys 6.2 us against 9.8, 512 keys 10.3 and 10.3, 1024 keys 14.4
// and 11.1.
//
// Over a grid of 1 - 32 sequences of 16 - 2048 keys, 64, 128 and 256 elements, bf16 and e4m3, 4 and 16 heads a key
// head, the rule takes the faster form, or one within 8 % of it, in 308 of 336 cases. It is off most for more pairs
// than SMs of 64 elements, of which an SM holds several blocks (256 pairs of 128 keys: two launches 9.8 us, one would
// take 6.2), and at its upper end for few pairs that two launches would split further (4 pairs of 512 keys with 16
// heads: one launch 12.3 us, two 8.8; 8 pairs with 4 heads 10.3 and 8.2; 256 elements in e4m3 14.9 and 11.1).
constexpr int kShortKeys = 64;
// Keys that a share has at least: below that its fixed costs weigh more than the loads that another warp would take
// over.
constexpr int kLeastKeys = 32;

int heads_per_unit(int group, int dim) { return group > 8 && dim <= 128 ? 16 : 8; }

// Calls f with the Shape of a call.
template <typename F>
auto with_shape(int dim, int group, int cache_type, F f) {
  auto heads = [&](auto d, auto mode) {
    constexpr int D = decltype(d)::value, M = decltype(mode)::value;
    if constexpr (D <= 128) {
      if (heads_per_unit(group, D) == 16) return f(Int<D>{}, Int<2>{}, Int<M>{});
    }
    return f(Int<D>{}, Int<1>{}, Int<M>{});
  };
  auto modes = [&](auto d) {
    return cache_type == ATTN_BF16  ? heads(d, Int<MODE_BF16>{})
           : cache_type == ATTN_F16 ? heads(d, Int<MODE_F16>{})
                                    : heads(d, Int<MODE_E4M3>{});
  };
  return dim == 64 ? modes(Int<64>{}) : dim == 96 ? modes(Int<96>{}) : dim == 128 ? modes(Int<128>{})
      : modes(Int<256>{});
}

int pairs_of(const Params &p) { return p.batch * p.kv_heads * p.chunks; }

// The lengths are on the device: what counts on the host is the most that they can be.
int longest_of(const Params &p) { return p.window > 0 ? std::min(p.window, p.capacity) : p.capacity; }

// A block for each pair, no more than SMs. From half the SMs on there is less to split: twice the keys (128 pairs of
// 1024 keys: 14.4 us against 18.2; of 2048, which take two launches: 24.7 and 26.9).
template <typename S>
bool is_short(const Params &p) {
  const int pairs = pairs_of(p), sms = device_sm_count();
  return pairs <= sms && longest_of(p) <= kShortKeys * S::kTeam * (2 * pairs > sms ? 2 : 1);
}

template <int D, int NT, int MODE, int GROUPS>
int launch_join(const Params &p, cudaStream_t s) {
  constexpr int kLanes = 256 / GROUPS;
  const dim3 grid(static_cast<unsigned>(pairs_of(p)), (Shape<D, NT, MODE>::kFrags * 32 + kLanes - 1) / kLanes);
  return launch_after(paged_join_kernel<D, NT, MODE, GROUPS>, grid, 256, s, p);
}

template <int D, int NT, int MODE>
int launch(Params p, cudaStream_t s) {
  using S = Shape<D, NT, MODE>;
  // The attribute belongs to the device's context: set once for each device.
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(paged_kernel<D, NT, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(paged_short_kernel<D, NT, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
        S::kTeam * S::kSmem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  p.blocks = device_sm_count() * S::kBlocks;
  p.least = kLeastKeys / S::kKeys;
  const int pairs = pairs_of(p);
  if (is_short<S>(p)) {
    paged_short_kernel<D, NT, MODE><<<pairs, 32 * S::kTeam, S::kTeam * S::kSmem, s>>>(p);
    return cudaGetLastError();
  }
  paged_kernel<D, NT, MODE><<<p.blocks, 32, S::kSmem, s>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (longest_of(p) <= S::kKeys) return 0;  // no pair has two tiles: nothing to join
  // Many parts of each of a few pairs are shared by eight sets of threads (8 pairs of 32768 keys, 148 parts: 35 us the
  // whole call, with one set 56); few parts of many pairs are not worth the exchange (512 pairs of 2048 keys: 68 us
  // with one set, 76 with eight). The two are level at 128 pairs for 128 elements (2048 keys: 26.8 and 26.5), so that
  // between 50 and 128 pairs, which have one set, eight would be up to a quarter faster (64 pairs of 2048 keys: 20.4
  // and 16.4).
  const int shares = p.blocks;
  return pairs > shares / 24 ? launch_join<D, NT, MODE, 1>(p, s) : launch_join<D, NT, MODE, 8>(p, s);
}

// The pairs' spans, in whole 16 bytes.
size_t span_bytes(const Params &p) { return (static_cast<size_t>(pairs_of(p)) + 1) / 2 * 16; }

bool refuse_call(const KvCacheArgs &c, const PagedAttentionArgs &a) {
  return (c.dim != 64 && c.dim != 96 && c.dim != 128 && c.dim != 256) || a.batch < 0 || a.heads < 1 || c.kv_heads < 1 ||
         a.heads % c.kv_heads || c.pages < 0 || c.page_shift < 0 || c.page_shift > 20 || a.window < 0
             || a.max_pages < 0 ||
         (static_cast<long long>(c.pages) * c.kv_heads << c.page_shift) > 0x7fffffffll ||
         static_cast<long long>(a.batch) * c.kv_heads * ((a.heads / c.kv_heads + 7) / 8) > 0x7fffffffll ||
         (static_cast<long long>(a.max_pages) << c.page_shift) > 0x7fffffffll - 256;
}

Params params_of(const KvCacheArgs &c, const PagedAttentionArgs &a) {
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
  p.capacity = c.pages > 0 ? a.max_pages << c.page_shift : 0;  // without pages there is not even an address to skip
  p.window = a.window;
  p.scale = a.scale;
  p.softcap = a.softcap;
  p.out = a.out;
  p.lse = a.lse;
  p.q_bf16 = a.q_type == ATTN_BF16;
  p.out_f32 = a.out_type == ATTN_F32;
  return p;
}

}  // namespace
}  // namespace attn

using namespace attn;

size_t paged_attention_workspace(const KvCacheArgs &c, const PagedAttentionArgs &a) {
  if (refuse_call(c, a)) return 0;
  const Params p = params_of(c, a);
  return with_shape(c.dim, p.group, c.type, [&](auto d, auto nt, auto mode) -> size_t {
    using S = Shape<decltype(d)::value, decltype(nt)::value, decltype(mode)::value>;
    return is_short<S>(p) ? 0 : span_bytes(p) + static_cast<size_t>(device_sm_count()) * S::kBlocks * 2 * S::kPart * 4;
  });
}

int paged_attention(const KvCacheArgs &c, const PagedAttentionArgs &a, void *workspace, size_t workspace_bytes,
    void *stream) {
  if (refuse_call(c, a) || (c.type == ATTN_E4M3 && c.pages > 0 && (!c.k_scale || !c.v_scale)) ||
      (a.q_type != ATTN_BF16 && a.q_type != ATTN_F16) || (c.type != ATTN_E4M3 && c.type != a.q_type) ||
      (a.out_type != a.q_type && a.out_type != ATTN_F32) || workspace_bytes < paged_attention_workspace(c, a)) {
    return cudaErrorInvalidValue;
  }
  if (a.batch == 0) return 0;
  Params p = params_of(c, a);
  // A warp counts its tiles (of 16 keys at least) in 32 bits.
  if (pairs_of(p) > 0x7fffffffll * device_sm_count() / (p.capacity / 16 + 1)) return cudaErrorInvalidValue;
  p.spans = static_cast<int2 *>(workspace);
  p.partial = reinterpret_cast<float *>(static_cast<char *>(workspace) + span_bytes(p));
  return with_shape(c.dim, p.group, c.type, [&](auto d, auto nt, auto mode) -> int {
    return launch<decltype(d)::value, decltype(nt)::value, decltype(mode)::value>(p, static_cast<cudaStream_t>(stream));
  });
}

}  // namespace kernels
}  // namespace rocshmem
