// Operators around attention that pass over their rows once: norm and rotation of query and key heads (forward and
// backward), writes into and reads from a paged cache, the join of partial attention results.
//
// All of them are bound by memory. A row (one head of one token) lies in 8, 16 or 32 neighbouring lanes, eight elements
// a lane; sums over a row by shuffles, nothing in shared memory but the weights' gradients. No counterpart exists in
// the reference.
#include "attention_common.cuh"

namespace rocshmem {
namespace kernels {

namespace attn {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ long long load_index(const void *p, int wide, int i) {
  return wide ? static_cast<const long long *>(p)[i] : static_cast<const int *>(p)[i];
}

// ---- norm and rotation -------------------------------------------------------------------------------------------

template <typename T, typename W>
struct NormRope {
  const T *q, *k;
  long long q_token, q_head, k_token, k_head;
  const W *q_weight, *k_weight;
  const void *positions;
  const float *table;
  int tokens, q_heads, k_heads, dim, rotary, table_rows;
  float eps, inv_dim;
  int wide_positions;
};

// The eight elements of a lane: two pieces of four, so that both elements of each of its pairs are among them and the
// rotation needs no exchange. Pairs (i, i + rotary / 2): the first lanes have a piece of either half, those behind
// eight neighbours that are not rotated. Pairs (2i, 2i + 1): eight neighbours.
template <bool INTERLEAVED>
struct Place {
  int e0, e1;
  bool in_row, rotated;
  __device__ __forceinline__ Place(int lane, int dim, int rotary) {
    in_row = 8 * lane < dim;
    rotated = 8 * lane < rotary;
    const bool halves = !INTERLEAVED && rotated;
    e0 = halves ? 4 * lane : 8 * lane;
    e1 = halves ? rotary / 2 + 4 * lane : 8 * lane + 4;
  }
};

template <typename T>
struct RawRow {
  Raw4<T> a, b;
};
template <typename T>
__device__ __forceinline__ void unpack(const RawRow<T> &r, float2 (&x)[4]) {
  unpack4(r.a, x);
  unpack4(r.b, x + 2);
}

// Cosines and sines of the lane's four pairs, as the packed products of rotate() take them.
template <bool INTERLEAVED>
struct Turn {
  float2 c[INTERLEAVED ? 4 : 2], s[INTERLEAVED ? 4 : 2];
  __device__ __forceinline__ void load(const float *row, int rotary, int lane) {
    const float4 cv = *reinterpret_cast<const float4 *>(row + 4 * lane);
    const float4 sv = *reinterpret_cast<const float4 *>(row + rotary / 2 + 4 * lane);
    if constexpr (INTERLEAVED) {
      c[0] = both(cv.x), c[1] = both(cv.y), c[2] = both(cv.z), c[3] = both(cv.w);
      s[0] = make_float2(-sv.x, sv.x), s[1] = make_float2(-sv.y, sv.y);
      s[2] = make_float2(-sv.z, sv.z), s[3] = make_float2(-sv.w, sv.w);
    } else {
      c[0] = make_float2(cv.x, cv.y), c[1] = make_float2(cv.z, cv.w);
      s[0] = make_float2(sv.x, sv.y), s[1] = make_float2(sv.z, sv.w);
    }
  }
};

// Rotates the lane's four pairs; BACK: the other way.
template <bool BACK, bool INTERLEAVED>
__device__ __forceinline__ void rotate(float2 (&x)[4], const Turn<INTERLEAVED> &a) {
#pragma unroll
  for (int i = 0; i < (INTERLEAVED ? 4 : 2); ++i) {
    if constexpr (INTERLEAVED) {  // (u, v) -> (u, v) c + (v, u) (-s, s)
      const float2 s = BACK ? make_float2(a.s[i].y, a.s[i].x) : a.s[i];
      x[i] = fma2(make_float2(x[i].y, x[i].x), s, mul2(x[i], a.c[i]));
    } else {
      const float2 n = make_float2(-a.s[i].x, -a.s[i].y), s = BACK ? n : a.s[i], ns = BACK ? a.s[i] : n;
      const float2 u = x[i], v = x[2 + i];
      x[i] = fma2(v, ns, mul2(u, a.c[i]));
      x[2 + i] = fma2(u, s, mul2(v, a.c[i]));
    }
  }
}

// ROWS heads of one token that a group of lanes takes at a time, all of queries or all of keys: their loads are issued
// before the first is used, and they share weights and angles.
template <typename T, typename W>
struct Side {
  const T *x;
  const W *weight;
  long long token, head;
  int heads;
  __device__ __forceinline__ Side(const NormRope<T, W> &a, bool is_q)
      : x(is_q ? a.q : a.k), weight(is_q ? a.q_weight : a.k_weight), token(is_q ? a.q_token : a.k_token),
        head(is_q ? a.q_head : a.k_head), heads(is_q ? a.q_heads : a.k_heads) {}
};

// 16384 tokens x (32 + 8) heads of 128, bf16: 61.5 us for 344 MB (5.6 TB/s; a device copy: 6.4), with two thirds of the
// issue slots and half of the integer pipe busy; fp32, 8192 tokens: 57 us for 340 MB (5.9). Four rows in flight and
// five blocks an SM, for which the 16-bit form with pairs of halves spills 16 - 20 bytes a thread; without spills, with
// four blocks, it takes 70 us, with three 69, with six, which spill more, 90; two rows 73, eight 65. One rounding: that
// of the result.
template <typename T, typename W, int LANES, int ROWS, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 3 : 5) norm_rope_kernel(NormRope<T, W> a, unsigned q_items,
    unsigned items, Divisor q_chunks, Divisor k_chunks, T *q_out, T *k_out) {
  const int lane = threadIdx.x % LANES;
  const Place<INTERLEAVED> at(lane, a.dim, a.rotary);
  // All lanes of a warp take part in every shuffle: groups past the last item have no rows.
  const unsigned mine = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const bool is_q = mine < q_items;
  const Side<T, W> side(a, is_q);
  const unsigned item = is_q ? mine : min(mine, items - 1) - q_items, t = divide(item, is_q ? q_chunks : k_chunks);
  const int h0 = (item - t * (is_q ? q_chunks.d : k_chunks.d)) * ROWS;
  const int left = mine < items && at.in_row ? side.heads - h0 : 0;
  const long long pos = load_index(a.positions, a.wide_positions, t);
  const T *const rows = side.x + t * side.token + h0 * side.head;
  RawRow<T> raw[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    raw[r] = RawRow<T>{};
    if (r < left) raw[r] = RawRow<T>{load4(rows + r * side.head + at.e0), load4(rows + r * side.head + at.e1)};
  }
  float2 w[4] = {};
  if (at.in_row) {
    unpack4(load4(side.weight + at.e0), w);
    unpack4(load4(side.weight + at.e1), w + 2);
  }
  const bool live = pos >= 0, known = pos < a.table_rows, turn = at.rotated && live && known;
  Turn<INTERLEAVED> angles;
  if (turn) angles.load(a.table + pos * a.rotary, a.rotary, lane);
  // A position without angles: NaN, not a wrong rotation.
  const float eps = known ? a.eps : __int_as_float(0x7fc00000);
  T *const out = (is_q ? q_out : k_out) + (static_cast<long long>(t) * side.heads + h0) * a.dim;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    float2 x[4];
    unpack(raw[r], x);
    float2 square = mul2(x[0], x[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) square = fma2(x[i], x[i], square);
    const float scale = rsqrtf(fmaf(group_sum<LANES>(square.x + square.y), a.inv_dim, eps));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = mul2(x[i], mul2(both(scale), w[i]));
    if (turn) rotate<false>(x, angles);
    if (!live) x[0] = x[1] = x[2] = x[3] = make_float2(0.f, 0.f);
    if (r < left) {
      store4(out + r * a.dim + at.e0, x);
      store4(out + r * a.dim + at.e1, x + 2);
    }
  }
}

// With g the gradient of the output rotated back, n = x r and a = w g: dx = r (a - n mean(a n)), dw = sum of g n. The
// norm is computed again (x is read anyway). Blocks below q_blocks have the queries, the others the keys, in
// proportion. Each group of lanes keeps the sums of its columns of the weight in registers over all its rows; a block
// adds those up in a fixed order, and norm_rope_weights_kernel adds the blocks' sums, so that the gradients are the
// same in every run.
//
// The case above: 101 us for 512 MB (5.1 TB/s), both kernels, without the host. 61 % of the issue slots; what is left
// is the latency of an item's position, then its angles. Two rows in flight and three blocks an SM: four rows 113, four
// blocks (spilling) 114, one row in four blocks 138; positions looked up an item ahead 115; items of eight heads 104;
// more blocks than fit at once 106 - 121.
template <typename T, typename W, int LANES, int ROWS, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 3) norm_rope_backward_kernel(NormRope<T, W> a, unsigned q_items,
    unsigned items, int q_blocks, const T *gq, const T *gk, T *dq, T *dk, float *partial) {
  extern __shared__ float sums[];  // [groups][dim]
  // The sum over the blocks may be set up from here on; it waits for the end of this grid before it reads.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  constexpr int kGroups = kThreads / LANES;
  const Place<INTERLEAVED> at(lane, a.dim, a.rotary);
  const bool is_q = static_cast<int>(blockIdx.x) < q_blocks;
  const Side<T, W> side(a, is_q);
  const unsigned n_items = is_q ? q_items : items - q_items, block = is_q ? blockIdx.x : blockIdx.x - q_blocks;
  const unsigned step = (is_q ? q_blocks : gridDim.x - q_blocks) * kGroups, chunks = (side.heads + ROWS - 1) / ROWS;
  const T *const grad = is_q ? gq : gk;
  T *const out = is_q ? dq : dk;
  float2 w[4] = {}, dw[4] = {};
  if (at.in_row) {
    unpack4(load4(side.weight + at.e0), w);
    unpack4(load4(side.weight + at.e1), w + 2);
  }
  // The same number of rounds for all groups of a block, for the shuffles; a group behind the last item has no rows.
  // Token and chunk move by the step's quotient and remainder.
  const unsigned start = block * kGroups + group, step_t = step / chunks, step_c = step - step_t * chunks;
  unsigned t = start / chunks, chunk = start - t * chunks;
  for (unsigned base = block * kGroups; base < n_items; base += step) {
    const bool has = base + group < n_items;
    const int h0 = chunk * ROWS, left = has && at.in_row ? side.heads - h0 : 0;
    const long long pos = load_index(a.positions, a.wide_positions, has ? t : 0);
    const T *const rows = side.x + t * side.token + h0 * side.head;
    const long long plain = (static_cast<long long>(t) * side.heads + h0) * a.dim;
    RawRow<T> raw[ROWS], graw[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      raw[r] = RawRow<T>{};
      graw[r] = RawRow<T>{};
      if (r < left) {
        const T *row = rows + r * side.head, *g = grad + plain + r * a.dim;
        raw[r] = RawRow<T>{load4(row + at.e0), load4(row + at.e1)};
        graw[r] = RawRow<T>{load4(g + at.e0), load4(g + at.e1)};
      }
    }
    const bool live = pos >= 0, known = pos < a.table_rows, turn = at.rotated && live && known;
    Turn<INTERLEAVED> angles;
    if (turn) angles.load(a.table + pos * a.rotary, a.rotary, lane);
    const float eps = known ? a.eps : __int_as_float(0x7fc00000);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float2 x[4], g[4];
      unpack(raw[r], x);
      unpack(graw[r], g);
      if (!live) {  // a padded token leaves nothing in the weights' gradients, whatever its rows hold
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = g[i] = make_float2(0.f, 0.f);
      }
      if (turn) rotate<true>(g, angles);
      float2 wg[4], square = mul2(x[0], x[0]), dots;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        wg[i] = mul2(g[i], w[i]);
        dots = i == 0 ? mul2(x[i], wg[i]) : fma2(x[i], wg[i], dots);
        if (i > 0) square = fma2(x[i], x[i], square);
      }
      const float sum = group_sum<LANES>(square.x + square.y), dot = group_sum<LANES>(dots.x + dots.y);
      // Rows that are not there add zeros: with their sum of zero and eps = 0 the scale would be infinite.
      const float scale = rsqrtf(r < side.heads - h0 && has && live ? fmaf(sum, a.inv_dim, eps) : 1.f);
      const float2 s2 = both(scale), mean = both(-dot * scale * a.inv_dim);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 n = mul2(x[i], s2);
        dw[i] = fma2(g[i], n, dw[i]);
        x[i] = mul2(s2, fma2(n, mean, wg[i]));
      }
      if (r < left) {
        T *to = out + plain + r * a.dim;
        store4(to + at.e0, x);
        store4(to + at.e1, x + 2);
      }
    }
    t += step_t;
    chunk += step_c;
    if (chunk >= chunks) {
      chunk -= chunks;
      ++t;
    }
  }
  if (at.in_row) {
    store4(sums + group * a.dim + at.e0, dw);
    store4(sums + group * a.dim + at.e1, dw + 2);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.dim; i += kThreads) {
    float v = 0.f;
    for (int g = 0; g < kGroups; ++g) v += sums[g * a.dim + i];
    partial[static_cast<long long>(blockIdx.x) * a.dim + i] = v;
  }
}

// Adds the blocks' sums: a block has 32 columns of one weight, its warps take the rows in turn.
template <typename W>
__global__ void __launch_bounds__(1024) norm_rope_weights_kernel(const float *partial, int q_rows, int rows, int dim,
    W *dq_weight, W *dk_weight) {
  __shared__ float s[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int col = blockIdx.x * 32 + threadIdx.x % 32, warp = threadIdx.x / 32;
  const int first = blockIdx.y ? q_rows : 0, end = blockIdx.y ? rows : q_rows;
  float v = 0.f;
  if (col < dim) {
#pragma unroll 4
    for (int r = first + warp; r < end; r += 32) v += partial[static_cast<long long>(r) * dim + col];
  }
  s[warp][threadIdx.x % 32] = v;
  __syncthreads();
  // Warp w adds the 32 sums of column w.
  const float x = group_sum<32>(s[threadIdx.x % 32][warp]);
  const int c = blockIdx.x * 32 + warp;
  if (threadIdx.x % 32 == 0 && c < dim) store1((blockIdx.y ? dk_weight : dq_weight) + c, x);
}

// ---- the paged cache ---------------------------------------------------------------------------------------------

template <typename C>
struct Cache {
  C *k, *v;
  float *k_scale, *v_scale;
  int slots;
  int kv_heads, shift, dim;
  Divisor each;  // two times kv_heads
};

// The head and the first of its tokens that a group of lanes has.
struct Row {
  long long token;
  int head;
  bool is_v;
};
// each: two times the heads
__device__ __forceinline__ Row row_of(unsigned group, int tokens_each, const Divisor &each) {
  const unsigned chunk = divide(group, each), h = group - chunk * each.d, heads = each.d / 2;
  return Row{static_cast<long long>(chunk) * tokens_each, static_cast<int>(h < heads ? h : h - heads), h >= heads};
}

// The cache rows of the group's tokens: lane r looks up token r and hands it to the others. All lanes of the warp call
// it.
template <int LANES, int ROWS, typename C>
__device__ __forceinline__ void look_up_rows(const C &c, const Row &w, const void *slots, int wide_slots, int tokens,
    int (&row)[ROWS]) {
  const int lane = threadIdx.x % LANES;
  int mine = -1;
  if (lane < ROWS && w.token + lane < tokens) {
    mine = slot_row(load_index(slots, wide_slots, static_cast<int>(w.token) + lane), c.slots, c.shift, c.kv_heads,
        w.head);
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) row[r] = __shfl_sync(0xffffffffu, mine, r, LANES);
}

// A group of lanes takes one head's row (of k or of v) of ROWS neighbouring tokens, their loads first. Neighbouring
// groups take the token's other heads: reads are contiguous across a block, and a head's rows go to neighbouring places
// of its page.
//
// e4m3: with m the largest magnitude of the row, codes are x * (448 / m) and the factor m / 448. m is held above
// 2^-110, below which 448 / m would overflow. The largest magnitude is that of the bits, so that a NaN or infinity
// becomes m, and with it the factor: such a row reads back as NaN. Rounding to 4 bits is what the cache is for; the
// factor is fp32.
//
// 32768 tokens x 8 heads of 128, bf16 to e4m3: 39 us for 204 MB (5.2 TB/s), bound by the integer pipe (68 % busy before
// a lane looked up a token's row for the others and divisions became multiplications, 42 us); to bf16 43 us for 269 MB
// (6.2 TB/s).
template <typename T, typename C, int LANES, int ROWS>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 4 : 6) kv_write_kernel(Cache<C> c, const T *k, const T *v,
    long long k_token, long long k_head, long long v_token, long long v_head, const void *slots, int wide_slots,
    int tokens) {
  constexpr bool kQuantize = sizeof(C) == 1;
  const int lane = threadIdx.x % LANES;
  const bool in_row = 8 * lane < c.dim;
  const Row w = row_of(blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES, ROWS, c.each);
  const T *from = (w.is_v ? v + w.head * v_head : k + w.head * k_head) + w.token * (w.is_v ? v_token : k_token);
  const long long step = w.is_v ? v_token : k_token;
  Raw8<T> raw[ROWS];
  int to[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    raw[r] = Raw8<T>{};
    if (in_row && w.token + r < tokens) raw[r] = load8(from + r * step, lane);
  }
  look_up_rows<LANES>(c, w, slots, wide_slots, tokens, to);
  C *const base = (w.is_v ? c.v : c.k) + 8 * lane;
  float *const scales = w.is_v ? c.v_scale : c.k_scale;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    float x[8];
    unpack8(raw[r], x);
    if constexpr (kQuantize) {
      const float top = group_top<LANES>(raw[r]);
      // the comparison fails for NaN too
      const float m = top < INFINITY ? fmaxf(top, 0x1p-110f) : __int_as_float(0x7fc00000);
      const float inv = 448.0f / m;
      if (to[r] >= 0) {
        if (in_row) {
          uint32_t codes[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 y = mul2(make_float2(x[2 * i], x[2 * i + 1]), both(inv));
            codes[i] = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
          }
          *reinterpret_cast<uint2 *>(base + static_cast<long long>(to[r]) * c.dim) =
              make_uint2(__byte_perm(codes[0], codes[1], 0x5410), __byte_perm(codes[2], codes[3], 0x5410));
        }
        if (lane == 0) scales[to[r]] = m * (1.0f / 448.0f);
      }
    } else {
      if (to[r] >= 0 && in_row) store8(base + static_cast<long long>(to[r]) * c.dim, x);
    }
  }
}

// 16381 tokens x 8 heads of 128, e4m3 to bf16: 18.5 us for 102 MB; 65536 tokens: 66 us for 407 MB (6.2 TB/s).
template <typename T, typename C, int LANES, int ROWS>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(Cache<C> c, T *k_out, T *v_out, const void *slots,
    int wide_slots, int tokens) {
  const int lane = threadIdx.x % LANES;
  const bool in_row = 8 * lane < c.dim;
  const Row w = row_of(blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES, ROWS, c.each);
  const C *base = w.is_v ? c.v : c.k;
  T *out = (w.is_v ? v_out : k_out) + (w.token * c.kv_heads + w.head) * c.dim + 8 * lane;
  const long long step = static_cast<long long>(c.kv_heads) * c.dim;
  Raw8<C> raw[ROWS];
  float factor[ROWS];
  int from[ROWS];
  look_up_rows<LANES>(c, w, slots, wide_slots, tokens, from);
  if (!in_row) return;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    raw[r] = Raw8<C>{};
    factor[r] = 0.f;
    if (from[r] >= 0) {
      raw[r] = load8(base + static_cast<long long>(from[r]) * c.dim, lane);
      if constexpr (sizeof(C) == 1) factor[r] = (w.is_v ? c.v_scale : c.k_scale)[from[r]];
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (w.token + r >= tokens) return;
    float x[8];
    unpack8(raw[r], x);
    if constexpr (sizeof(C) == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 y = mul2(make_float2(x[2 * i], x[2 * i + 1]), both(factor[r]));
        x[2 * i] = y.x, x[2 * i + 1] = y.y;
      }
    }
    store8(out + r * step, x);
  }
}

// ---- the join of partial results ---------------------------------------------------------------------------------

// out = sum w_i o_i / sum w_i with w_i = exp(lse_i - max). A part whose lse is -inf has seen nothing and does not
// count, whatever its rows hold. Eight parts of 512 x 64 rows of 128 in fp32: 26.6 us for 144 MB (5.4 TB/s), bound by
// the memory's latency; the first parts' loads are on their way while the maximum is found.
template <typename T, typename O, int LANES>
__global__ void __launch_bounds__(kThreads) join_kernel(const T *outs, const float *lses, long long out_part,
    long long lse_part, int parts, long long rows, int dim, O *out, float *lse) {
  constexpr int kAhead = sizeof(T) == 4 ? 4 : 8;  // parts whose loads are in flight
  const int lane = threadIdx.x % LANES;
  const long long row = static_cast<long long>(blockIdx.x) * (kThreads / LANES) + threadIdx.x / LANES;
  if (row >= rows) return;
  const bool in_row = 8 * lane < dim;
  const T *from = outs + row * dim;
  Raw8<T> raw[kAhead];
  auto fetch = [&](int p0) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      raw[i] = Raw8<T>{};
      if (p0 + i < parts && in_row) raw[i] = load8(from + (p0 + i) * out_part, lane);
    }
  };
  fetch(0);  // on their way while the maximum is found
  float top = -INFINITY;
  bool bad = false;
#pragma unroll 4
  for (int p = 0; p < parts; ++p) {
    const float l = lses[p * lse_part + row];
    bad |= l != l;
    top = fmaxf(top, l);
  }
  const float base = top == -INFINITY ? 0.f : top;
  float acc[8] = {}, total = 0.f;
  for (int p0 = 0;;) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (p0 + i >= parts) break;
      const float l = lses[(p0 + i) * lse_part + row], w = expf(l - base);
      total += w;
      if (l == -INFINITY) continue;
      float x[8];
      unpack8(raw[i], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, x[e], acc[e]);
    }
    p0 += kAhead;
    if (p0 >= parts) break;
    fetch(p0);
  }
  const float inv = total > 0.f || bad ? 1.f / total : 0.f;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = acc[e] * inv;
  if (in_row) store8(out + row * dim + 8 * lane, x);
  if (lane == 0 && lse != nullptr) {
    lse[row] = bad ? __int_as_float(0x7fc00000) : total > 0.f ? base + logf(total) : -INFINITY;
  }
}

// ---- choice of the instantiation ---------------------------------------------------------------------------------

template <typename T>
struct Tag {
  using type = T;
};

template <typename F>
int with_type(int code, F f) {
  switch (code) {
    case ATTN_BF16: return f(Tag<__nv_bfloat16>{});
    case ATTN_F16: return f(Tag<__half>{});
    case ATTN_F32: return f(Tag<float>{});
    default: return cudaErrorInvalidValue;
  }
}

template <typename F>
int with_lanes(int dim, F f) {
  switch (row_lanes(dim)) {
    case 8: return f(Int<8>{});
    case 16: return f(Int<16>{});
    default: return f(Int<32>{});
  }
}

bool bad_rows(int dim) { return dim < 8 || dim > 256 || dim % 8; }

// Blocks of a launch with one group of lanes for each of `items`; 0 when the kernels could not number the groups in 32
// bits.
unsigned blocks_for(long long items, int lanes) {
  const long long per = kThreads / lanes, n = (items + per - 1) / per;
  return n * per > 0x7fffffffll ? 0u : static_cast<unsigned>(n);
}

// Groups of lanes that the GPU's SMs hold at once.
long long groups_at_once(int lanes) { return static_cast<long long>(device_sm_count()) * (2048 / lanes); }

// Items of `rows` heads.
long long items_of(int tokens, int heads, int rows) {
  return static_cast<long long>(tokens) * ((heads + rows - 1) / rows);
}

int backward_blocks() { return device_sm_count() * 3; }

template <typename T, typename W>
NormRope<T, W> norm_rope_args(const NormRopeArgs &a) {
  return NormRope<T, W>{static_cast<const T *>(a.q), static_cast<const T *>(a.k), a.q_token, a.q_head, a.k_token,
      a.k_head, static_cast<const W *>(a.q_weight), static_cast<const W *>(a.k_weight), a.positions, a.table, a.tokens,
      a.q_heads, a.k_heads, a.dim, a.rotary, a.table_rows, a.eps, 1.f / static_cast<float>(a.dim), a.wide_positions};
}

// The weights have the rows' type or fp32.
template <typename F>
int with_row_and_weight(const NormRopeArgs &a, F f) {
  if (a.weight_type != a.type && a.weight_type != ATTN_F32) return cudaErrorInvalidValue;
  return with_type(a.type, [&](auto t) -> int {
    using T = typename decltype(t)::type;
    return a.weight_type == ATTN_F32 ? f(Tag<T>{}, Tag<float>{}) : f(Tag<T>{}, Tag<T>{});
  });
}

bool refuse(const NormRopeArgs &a) {
  return bad_rows(a.dim) || a.rotary < 16 || a.rotary > a.dim || a.rotary % 16 || a.tokens < 0 || a.q_heads < 1 ||
         a.k_heads < 1 || a.table_rows < 1;
}

template <typename F>
int with_cache(const KvCacheArgs &c, F f) {
  auto args = [&](auto tag) {
    using C = typename decltype(tag)::type;
    return Cache<C>{static_cast<C *>(c.k), static_cast<C *>(c.v), c.k_scale, c.v_scale, c.pages << c.page_shift,
        c.kv_heads, c.page_shift, c.dim, divisor(2 * static_cast<uint32_t>(c.kv_heads))};
  };
  switch (c.type) {
    case ATTN_BF16: return f(args(Tag<__nv_bfloat16>{}), Tag<__nv_bfloat16>{});
    case ATTN_F16: return f(args(Tag<__half>{}), Tag<__half>{});
    case ATTN_E4M3: return f(args(Tag<e4m3>{}), Tag<e4m3>{});
    default: return cudaErrorInvalidValue;
  }
}

bool refuse(const KvCacheArgs &c) {
  return bad_rows(c.dim) || c.pages < 0 || c.kv_heads < 1 || c.page_shift < 0 || c.page_shift > 20 ||
         (static_cast<long long>(c.pages) * c.kv_heads << c.page_shift) > 0x7fffffffll ||
         (c.type == ATTN_E4M3 && c.pages > 0 && (!c.k_scale || !c.v_scale));
}

}  // namespace
}  // namespace attn

using namespace attn;

int qk_norm_rope(const NormRopeArgs &a, void *q_out, void *k_out, void *stream) {
  if (refuse(a)) return cudaErrorInvalidValue;
  if (a.tokens == 0) return 0;
  return with_row_and_weight(a, [&](auto t, auto w) -> int {
    using T = typename decltype(t)::type;
    using W = typename decltype(w)::type;
    return with_lanes(a.dim, [&](auto l) -> int {
      constexpr int kLanes = decltype(l)::value;
      auto launch = [&](auto rows, auto pairs) -> int {
        constexpr int kRows = decltype(rows)::value;
        const long long q_items = items_of(a.tokens, a.q_heads, kRows);
        const long long items = q_items + items_of(a.tokens, a.k_heads, kRows);
        const unsigned blocks = blocks_for(items, kLanes);
        if (!blocks) return cudaErrorInvalidValue;
        norm_rope_kernel<T, W, kLanes, kRows, decltype(pairs)::value != 0>
            <<<blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
                norm_rope_args<T, W>(a), static_cast<unsigned>(q_items), static_cast<unsigned>(items),
                divisor((a.q_heads + kRows - 1) / kRows), divisor((a.k_heads + kRows - 1) / kRows),
                static_cast<T *>(q_out), static_cast<T *>(k_out));
        return cudaGetLastError();
      };
      // One row a group while that leaves SMs without work, four rows in flight beyond.
      const bool few = static_cast<long long>(a.tokens) * (a.q_heads + a.k_heads) <= groups_at_once(kLanes);
      if (a.interleaved) return few ? launch(Int<1>{}, Int<1>{}) : launch(Int<4>{}, Int<1>{});
      return few ? launch(Int<1>{}, Int<0>{}) : launch(Int<4>{}, Int<0>{});
    });
  });
}

size_t qk_norm_rope_workspace(int dim) { return static_cast<size_t>(backward_blocks()) * static_cast<size_t>(dim); }

int qk_norm_rope_backward(const NormRopeArgs &a, const void *gq, const void *gk, void *dq, void *dk, void *dq_weight,
    void *dk_weight, float *workspace, void *stream) {
  if (refuse(a)) return cudaErrorInvalidValue;
  return with_row_and_weight(a, [&](auto t, auto w) -> int {
    using T = typename decltype(t)::type;
    using W = typename decltype(w)::type;
    return with_lanes(a.dim, [&](auto l) -> int {
      constexpr int kLanes = decltype(l)::value;
      constexpr int kRows = 2;
      const cudaStream_t s = static_cast<cudaStream_t>(stream);
      const long long q_items = items_of(a.tokens, a.q_heads, kRows);
      const long long items = q_items + items_of(a.tokens, a.k_heads, kRows);
      const long long per = kThreads / kLanes;
      if (items > 0x7fffffffll - backward_blocks() * per) return cudaErrorInvalidValue;
      // Blocks in proportion to the items of queries and keys, at least one for either.
      const long long wanted = std::min<long long>(backward_blocks(), (items + per - 1) / per);
      const int blocks = static_cast<int>(std::max<long long>(2, wanted));
      const long long q_share = q_items * blocks / std::max(items, 1ll);
      const int q_blocks = static_cast<int>(std::min<long long>(std::max<long long>(q_share, 1), blocks - 1));
      auto launch = [&](auto pairs) -> int {
        norm_rope_backward_kernel<T, W, kLanes, kRows, decltype(pairs)::value != 0>
            <<<blocks, kThreads, kThreads / kLanes * a.dim * sizeof(float), s>>>(
                norm_rope_args<T, W>(a), static_cast<unsigned>(q_items), static_cast<unsigned>(items), q_blocks,
                static_cast<const T *>(gq), static_cast<const T *>(gk), static_cast<T *>(dq), static_cast<T *>(dk),
                workspace);
        return cudaGetLastError();
      };
      const int e = a.interleaved ? launch(Int<1>{}) : launch(Int<0>{});
      if (e != cudaSuccess) return e;
      return launch_after(norm_rope_weights_kernel<W>, dim3((a.dim + 31) / 32, 2), 1024, s, workspace, q_blocks, blocks,
          a.dim, static_cast<W *>(dq_weight), static_cast<W *>(dk_weight));
    });
  });
}

int kv_cache_write(const KvCacheArgs &c, const void *k, const void *v, long long k_token, long long k_head,
    long long v_token, long long v_head, const void *slots, int wide_slots, int tokens, int type, void *stream) {
  if (refuse(c) || tokens < 0) return cudaErrorInvalidValue;
  if (tokens == 0) return 0;
  return with_type(type, [&](auto t) -> int {
    using T = typename decltype(t)::type;
    return with_cache(c, [&](auto cache, auto tag) -> int {
      using C = typename decltype(tag)::type;
      return with_lanes(c.dim, [&](auto l) -> int {
        constexpr int kLanes = decltype(l)::value;
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        const long long rows = static_cast<long long>(tokens) * 2 * c.kv_heads;
        auto launch = [&](auto n) -> int {
          constexpr int kRows = decltype(n)::value;
          const unsigned blocks = blocks_for((static_cast<long long>(tokens) + kRows - 1) / kRows * 2 * c.kv_heads,
              kLanes);
          if (!blocks) return cudaErrorInvalidValue;
          kv_write_kernel<T, C, kLanes, kRows><<<blocks, kThreads, 0, s>>>(
              cache, static_cast<const T *>(k), static_cast<const T *>(v), k_token, k_head, v_token, v_head, slots,
              wide_slots, tokens);
          return cudaGetLastError();
        };
        return rows <= groups_at_once(kLanes) ? launch(Int<1>{}) : launch(Int<4>{});
      });
    });
  });
}

int kv_cache_read(const KvCacheArgs &c, void *k_out, void *v_out, const void *slots, int wide_slots, int tokens,
    int type, void *stream) {
  if (refuse(c) || tokens < 0) return cudaErrorInvalidValue;
  if (tokens == 0) return 0;
  return with_type(type, [&](auto t) -> int {
    using T = typename decltype(t)::type;
    return with_cache(c, [&](auto cache, auto tag) -> int {
      using C = typename decltype(tag)::type;
      return with_lanes(c.dim, [&](auto l) -> int {
        constexpr int kLanes = decltype(l)::value;
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        const long long rows = static_cast<long long>(tokens) * 2 * c.kv_heads;
        auto launch = [&](auto n) -> int {
          constexpr int kRows = decltype(n)::value;
          const unsigned blocks = blocks_for((static_cast<long long>(tokens) + kRows - 1) / kRows * 2 * c.kv_heads,
              kLanes);
          if (!blocks) return cudaErrorInvalidValue;
          kv_read_kernel<T, C, kLanes, kRows><<<blocks, kThreads, 0, s>>>(cache, static_cast<T *>(k_out),
              static_cast<T *>(v_out), slots, wide_slots, tokens);
          return cudaGetLastError();
        };
        return rows <= groups_at_once(kLanes) ? launch(Int<1>{}) : launch(Int<4>{});
      });
    });
  });
}

int attention_join(const void *outs, const float *lses, long long out_part, long long lse_part, int parts,
    long long rows, int dim, int in_type, int out_type, void *out, float *lse, void *stream) {
  if (bad_rows(dim) || parts < 1 || rows < 0) return cudaErrorInvalidValue;
  if (rows == 0) return 0;
  return with_type(in_type, [&](auto t) -> int {
    using T = typename decltype(t)::type;
    return with_type(out_type, [&](auto o) -> int {
      using O = typename decltype(o)::type;
      return with_lanes(dim, [&](auto l) -> int {
        constexpr int kLanes = decltype(l)::value;
        const unsigned blocks = blocks_for(rows, kLanes);
        if (!blocks) return cudaErrorInvalidValue;
        join_kernel<T, O, kLanes><<<blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T *>(outs), lses, out_part, lse_part, parts, rows, dim, static_cast<O *>(out), lse);
        return cudaGetLastError();
      });
    });
  });
}

}  // namespace kernels
}  // namespace rocshmem
