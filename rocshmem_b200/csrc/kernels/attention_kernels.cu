// Operators around attention that pass over their rows once: norm and rotation of query and key heads (forward and
// backward), writes into and reads from a paged cache, the join of partial attention results.
//
// All of them are bound by memory. A row (one head of one token) lies in 8, 16 or 32 neighbouring lanes, eight elements a
// lane: 16-byte accesses for 16-bit types, sums over a row by shuffles, nothing in shared memory but the weights' gradients.
// No counterpart exists in the reference.
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

// What a lane needs of its token's position: cosines and sines for its eight elements.
struct Angles {
  float c[8], s[8];
};

// `lane` is the lane's place in its row, elements [8 lane, 8 lane + 8). Pairs are (i, i + rotary / 2), or (2i, 2i + 1).
__device__ __forceinline__ void load_angles(Angles &a, const float *row, int rotary, int lane, bool interleaved) {
  const int half = rotary / 2;
  if (interleaved) {
    const float4 c = *reinterpret_cast<const float4 *>(row + 4 * lane);
    const float4 s = *reinterpret_cast<const float4 *>(row + half + 4 * lane);
    const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a.c[i] = cv[i / 2];
      a.s[i] = i % 2 ? sv[i / 2] : -sv[i / 2];
    }
  } else {
    const int at = 8 * lane < half ? 8 * lane : 8 * lane - half;
    const float sign = 8 * lane < half ? -1.f : 1.f;
    unpack8(load8(row + at), a.c);
    unpack8(load8(row + half + at), a.s);
#pragma unroll
    for (int i = 0; i < 8; ++i) a.s[i] *= sign;
  }
}

// The other element of each of the lane's pairs. All lanes of the warp call it.
template <int LANES>
__device__ __forceinline__ void partners(const float (&y)[8], float (&other)[8], int rotary, int lane, bool interleaved) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) other[i] = y[i ^ 1];
  } else {
    const int half = rotary / 16;  // in lanes
    const int from = lane < half ? lane + half : lane < 2 * half ? lane - half : lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(0xffffffffu, y[i], from, LANES);
  }
}

template <typename T, typename W>
struct NormRope {
  const T *q, *k;
  long long q_token, q_head, k_token, k_head;
  const W *q_weight, *k_weight;
  const void *positions;
  const float *table;
  int tokens, q_heads, k_heads, dim, rotary, table_rows;
  float eps;
  int interleaved, wide_positions;
};

// Rows are taken ROWS at a time: an item is ROWS heads of one token, whose loads are all issued before the first is used
// and which share the token's angles.
template <typename T, typename W, int LANES, int ROWS>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(NormRope<T, W> a, T *q_out, T *k_out) {
  const int lane = threadIdx.x % LANES;
  const int heads = a.q_heads + a.k_heads;
  const unsigned chunks = (heads + ROWS - 1) / ROWS, items = a.tokens * chunks;
  // All lanes of a warp take part in every shuffle: groups past the last item work on it again and store nothing.
  const unsigned mine = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const unsigned item = min(mine, items - 1), t = item / chunks;
  const int h0 = (item - t * chunks) * ROWS;
  const bool in_row = 8 * lane < a.dim;
  const long long pos = load_index(a.positions, a.wide_positions, t);
  const bool live = pos >= 0, known = pos < a.table_rows;

  Raw8<T> raw[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int h = h0 + r;
    raw[r] = Raw8<T>{};
    if (live && in_row && h < heads) {
      raw[r] = load8(h < a.q_heads ? a.q + t * a.q_token + h * a.q_head : a.k + t * a.k_token + (h - a.q_heads) * a.k_head, lane);
    }
  }
  Angles ang;
  const bool rotated = 8 * lane < a.rotary;
  if (rotated && live && known) {
    load_angles(ang, a.table + pos * a.rotary, a.rotary, lane, a.interleaved);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) ang.c[i] = 1.f, ang.s[i] = 0.f;
  }
  float wq[8] = {}, wk[8] = {};
  if (in_row) {
    unpack8(load8(a.q_weight, lane), wq);
    unpack8(load8(a.k_weight, lane), wk);
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int h = h0 + r;
    float x[8], other[8], sum = 0.f;
    unpack8(raw[r], x);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
    sum = group_sum<LANES>(sum);
    float scale = rsqrtf(sum / static_cast<float>(a.dim) + a.eps);
    if (!known) scale = __int_as_float(0x7fc00000);  // a position without angles: NaN, not a wrong rotation
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= scale * (h < a.q_heads ? wq[i] : wk[i]);
    partners<LANES>(x, other, a.rotary, lane, a.interleaved);
    if (rotated) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fmaf(other[i], ang.s[i], x[i] * ang.c[i]);
    }
    if (!live) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
    }
    if (mine < items && in_row && h < heads) {
      T *to = h < a.q_heads ? q_out + (static_cast<long long>(t) * a.q_heads + h) * a.dim
                            : k_out + (static_cast<long long>(t) * a.k_heads + (h - a.q_heads)) * a.dim;
      store8(to + 8 * lane, x);
    }
  }
}

// With g the gradient of the output rotated back, n = x r and a = w g: dx = r (a - n mean(a n)), dw = sum of g n. The norm
// is computed again (x is read anyway). Each group of lanes keeps the sums of its columns of both weights in registers
// over all its rows; blocks add theirs up in a fixed order, and norm_rope_weights_kernel adds the blocks' sums, so that
// the gradients are the same in every run.
template <typename T, typename W, int LANES, int ROWS>
__global__ void __launch_bounds__(kThreads) norm_rope_backward_kernel(NormRope<T, W> a, const T *gq, const T *gk, T *dq,
                                                                      T *dk, float *partial) {
  extern __shared__ float sums[];  // [groups][2 * dim]
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  constexpr int kGroups = kThreads / LANES;
  const int heads = a.q_heads + a.k_heads;
  const unsigned chunks = (heads + ROWS - 1) / ROWS, items = a.tokens * chunks;
  const bool in_row = 8 * lane < a.dim, rotated = 8 * lane < a.rotary;
  float wq[8] = {}, wk[8] = {}, dwq[8] = {}, dwk[8] = {};
  if (in_row) {
    unpack8(load8(a.q_weight, lane), wq);
    unpack8(load8(a.k_weight, lane), wk);
  }
  const unsigned step = gridDim.x * kGroups;
  // The same number of rounds for all groups of a block, for the shuffles.
  for (unsigned base = blockIdx.x * kGroups; base < items; base += step) {
    const bool has = base + group < items;
    const unsigned item = has ? base + group : items - 1, t = item / chunks;
    const int h0 = (item - t * chunks) * ROWS;
    const long long pos = load_index(a.positions, a.wide_positions, t);
    const bool live = pos >= 0, known = pos < a.table_rows;
    Raw8<T> raw[ROWS], graw[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int h = h0 + r;
      raw[r] = Raw8<T>{};
      graw[r] = Raw8<T>{};
      if (has && live && in_row && h < heads) {
        const bool is_q = h < a.q_heads;
        raw[r] = load8(is_q ? a.q + t * a.q_token + h * a.q_head : a.k + t * a.k_token + (h - a.q_heads) * a.k_head, lane);
        graw[r] = load8(is_q ? gq + (static_cast<long long>(t) * a.q_heads + h) * a.dim
                             : gk + (static_cast<long long>(t) * a.k_heads + (h - a.q_heads)) * a.dim, lane);
      }
    }
    Angles ang;
    if (rotated && live && known) {
      load_angles(ang, a.table + pos * a.rotary, a.rotary, lane, a.interleaved);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) ang.c[i] = 1.f, ang.s[i] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int h = h0 + r;
      const bool is_q = h < a.q_heads;
      float x[8], g[8], other[8], sum = 0.f, dot = 0.f;
      unpack8(raw[r], x);
      unpack8(graw[r], g);
      partners<LANES>(g, other, a.rotary, lane, a.interleaved);
      if (rotated) {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = fmaf(other[i], -ang.s[i], g[i] * ang.c[i]);  // the inverse rotation
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum = fmaf(x[i], x[i], sum);
        dot = fmaf(x[i], g[i] * (is_q ? wq[i] : wk[i]), dot);
      }
      sum = group_sum<LANES>(sum);
      dot = group_sum<LANES>(dot);
      float scale = rsqrtf(sum / static_cast<float>(a.dim) + a.eps);
      if (!known) scale = __int_as_float(0x7fc00000);
      const float mean = dot * scale / static_cast<float>(a.dim);
      if (live) {  // a padded token leaves nothing in the weights' gradients, whatever its gradient holds
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float n = x[i] * scale;
          if (is_q) dwq[i] = fmaf(g[i], n, dwq[i]);
          else dwk[i] = fmaf(g[i], n, dwk[i]);
          d[i] = scale * (g[i] * (is_q ? wq[i] : wk[i]) - n * mean);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = d[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.f;
      }
      if (has && in_row && h < heads) {
        T *to = is_q ? dq + (static_cast<long long>(t) * a.q_heads + h) * a.dim
                     : dk + (static_cast<long long>(t) * a.k_heads + (h - a.q_heads)) * a.dim;
        store8(to + 8 * lane, x);
      }
    }
  }
  if (in_row) {
    store8(sums + group * 2 * a.dim + 8 * lane, dwq);
    store8(sums + group * 2 * a.dim + a.dim + 8 * lane, dwk);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.dim; i += kThreads) {
    float v = 0.f;
    for (int g = 0; g < kGroups; ++g) v += sums[g * 2 * a.dim + i];
    partial[static_cast<long long>(blockIdx.x) * 2 * a.dim + i] = v;
  }
}

// Adds the blocks' sums: a block has 32 columns, its warps take the rows in turn.
template <typename W>
__global__ void __launch_bounds__(1024) norm_rope_weights_kernel(const float *partial, int rows, int dim, W *dq_weight,
                                                                 W *dk_weight) {
  __shared__ float s[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x % 32, warp = threadIdx.x / 32;
  float v = 0.f;
  if (col < 2 * dim) {
    for (int r = warp; r < rows; r += 32) v += partial[static_cast<long long>(r) * 2 * dim + col];
  }
  s[warp][threadIdx.x % 32] = v;
  __syncthreads();
  // Warp w adds the 32 sums of column w.
  float x = s[threadIdx.x % 32][warp];
  x = group_sum<32>(x);
  const int c = blockIdx.x * 32 + warp;
  if (threadIdx.x % 32 == 0 && c < 2 * dim) store1(c < dim ? dq_weight + c : dk_weight + (c - dim), x);
}

// ---- the paged cache ---------------------------------------------------------------------------------------------

template <typename C>
struct Cache {
  C *k, *v;
  float *k_scale, *v_scale;
  long long slots;
  int kv_heads, shift, dim;
};

// The head and the first of its tokens that a group of lanes has.
struct Row {
  long long token;
  int head;
  bool is_v;
};
__device__ __forceinline__ Row row_of(unsigned group, int tokens_each, int kv_heads) {
  const unsigned each = 2 * kv_heads, chunk = group / each, h = group - chunk * each;
  return Row{static_cast<long long>(chunk) * tokens_each, static_cast<int>(h < kv_heads ? h : h - kv_heads), h >= kv_heads};
}

// A group of lanes takes one head's row (of k or of v) of ROWS neighbouring tokens, their loads first. Neighbouring groups
// take the token's other heads: reads are contiguous across a block, and a head's rows go to neighbouring places of its page.
//
// e4m3: with m the largest magnitude of the row, codes are x * (448 / m) and the factor m / 448. m is held above 2^-110,
// below which 448 / m would overflow. The largest magnitude is that of the bits, so that a NaN or infinity becomes m, and
// with it the factor: such a row reads back as NaN.
template <typename T, typename C, int LANES, int ROWS>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(Cache<C> c, const T *k, const T *v, long long k_token,
                                                            long long k_head, long long v_token, long long v_head,
                                                            const void *slots, int wide_slots, int tokens) {
  constexpr bool kQuantize = sizeof(C) == 1;
  const int lane = threadIdx.x % LANES;
  const bool in_row = 8 * lane < c.dim;
  const Row w = row_of(blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES, ROWS, c.kv_heads);
  const T *from = (w.is_v ? v + w.head * v_head : k + w.head * k_head) + w.token * (w.is_v ? v_token : k_token);
  const long long step = w.is_v ? v_token : k_token;
  Raw8<T> raw[ROWS];
  long long to[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    to[r] = -1;
    raw[r] = Raw8<T>{};
    if (w.token + r < tokens) {
      if (in_row) raw[r] = load8(from + r * step, lane);
      to[r] = slot_row(load_index(slots, wide_slots, static_cast<int>(w.token) + r), c.slots, c.shift, c.kv_heads, w.head);
    }
  }
  C *base = w.is_v ? c.v : c.k;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    float x[8];
    unpack8(raw[r], x);
    if constexpr (kQuantize) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
      top = group_max<LANES>(top);
      float m = __uint_as_float(max(top, __float_as_uint(0x1p-110f)));
      if (top >= 0x7f800000u) m = __int_as_float(0x7fc00000);
      const float inv = 448.0f / m;
      if (to[r] >= 0) {
        if (in_row) {
          uint2 o;
          uint32_t *codes = reinterpret_cast<uint32_t *>(&o);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 a = make_float2(x[4 * i] * inv, x[4 * i + 1] * inv);
            const float2 b = make_float2(x[4 * i + 2] * inv, x[4 * i + 3] * inv);
            codes[i] = __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3) |
                   static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3)) << 16;
          }
          *reinterpret_cast<uint2 *>(base + to[r] * c.dim + 8 * lane) = o;
        }
        if (lane == 0) (w.is_v ? c.v_scale : c.k_scale)[to[r]] = m * (1.0f / 448.0f);
      }
    } else {
      if (to[r] >= 0 && in_row) store8(base + to[r] * c.dim + 8 * lane, x);
    }
  }
}

template <typename T, typename C, int LANES, int ROWS>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(Cache<C> c, T *k_out, T *v_out, const void *slots,
                                                           int wide_slots, int tokens) {
  const int lane = threadIdx.x % LANES;
  const bool in_row = 8 * lane < c.dim;
  const Row w = row_of(blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES, ROWS, c.kv_heads);
  const C *base = w.is_v ? c.v : c.k;
  T *out = (w.is_v ? v_out : k_out) + (w.token * c.kv_heads + w.head) * c.dim + 8 * lane;
  const long long step = static_cast<long long>(c.kv_heads) * c.dim;
  if (!in_row) return;
  Raw8<C> raw[ROWS];
  float factor[ROWS];
  long long from[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    from[r] = w.token + r < tokens ? slot_row(load_index(slots, wide_slots, static_cast<int>(w.token) + r), c.slots, c.shift,
                                              c.kv_heads, w.head) : -1;
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    raw[r] = Raw8<C>{};
    factor[r] = 0.f;
    if (from[r] >= 0) {
      raw[r] = load8(base + from[r] * c.dim, lane);
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
      for (int i = 0; i < 8; ++i) x[i] *= factor[r];
    }
    store8(out + r * step, x);
  }
}

// ---- the join of partial results ---------------------------------------------------------------------------------

// out = sum w_i o_i / sum w_i with w_i = exp(lse_i - max). A part whose lse is -inf has seen nothing and
// does not count, whatever its rows hold.
template <typename T, typename O, int LANES>
__global__ void __launch_bounds__(kThreads) join_kernel(const T *outs, const float *lses, long long out_part,
                                                        long long lse_part, int parts, long long rows, int dim, O *out,
                                                        float *lse) {
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
  if (lane == 0 && lse != nullptr) lse[row] = bad ? __int_as_float(0x7fc00000) : total > 0.f ? base + logf(total) : -INFINITY;
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

// Blocks of a launch with one group of lanes for each of `items`; 0 when the kernels could not number the groups in 32 bits.
unsigned blocks_for(long long items, int lanes) {
  const long long per = kThreads / lanes, n = (items + per - 1) / per;
  return n * per > 0x7fffffffll ? 0u : static_cast<unsigned>(n);
}

int backward_blocks() { return device_sm_count() * 2; }

template <typename T, typename W>
NormRope<T, W> norm_rope_args(const NormRopeArgs &a) {
  return NormRope<T, W>{static_cast<const T *>(a.q), static_cast<const T *>(a.k), a.q_token, a.q_head, a.k_token, a.k_head,
                        static_cast<const W *>(a.q_weight), static_cast<const W *>(a.k_weight), a.positions, a.table,
                        a.tokens, a.q_heads, a.k_heads, a.dim, a.rotary, a.table_rows, a.eps, a.interleaved,
                        a.wide_positions};
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
  return bad_rows(a.dim) || a.rotary < 16 || a.rotary > a.dim || a.rotary % 16 || a.tokens < 0 || a.q_heads < 0 ||
         a.k_heads < 0 || a.q_heads + a.k_heads < 1 || a.table_rows < 1;
}

template <typename F>
int with_cache(const KvCacheArgs &c, F f) {
  auto args = [&](auto tag) {
    using C = typename decltype(tag)::type;
    return Cache<C>{static_cast<C *>(c.k), static_cast<C *>(c.v), c.k_scale, c.v_scale,
                    static_cast<long long>(c.pages) << c.page_shift, c.kv_heads, c.page_shift, c.dim};
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
         (c.type == ATTN_E4M3 && (!c.k_scale || !c.v_scale));
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
      const auto args = norm_rope_args<T, W>(a);
      const cudaStream_t s = static_cast<cudaStream_t>(stream);
      const int heads = a.q_heads + a.k_heads;
      auto launch = [&](auto rows) -> int {
        constexpr int kRows = decltype(rows)::value;
        const unsigned blocks = blocks_for(static_cast<long long>(a.tokens) * ((heads + kRows - 1) / kRows), kLanes);
        if (!blocks) return cudaErrorInvalidValue;
        norm_rope_kernel<T, W, kLanes, kRows><<<blocks, kThreads, 0, s>>>(args, static_cast<T *>(q_out), static_cast<T *>(k_out));
        return cudaGetLastError();
      };
      // One row a group while that leaves SMs without work, four rows in flight beyond.
      const long long groups = static_cast<long long>(device_sm_count()) * (2048 / kLanes);
      return static_cast<long long>(a.tokens) * heads <= groups ? launch(Int<1>{}) : launch(Int<4>{});
    });
  });
}

size_t qk_norm_rope_workspace(int dim) { return static_cast<size_t>(backward_blocks()) * 2 * static_cast<size_t>(dim); }

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
      const int heads = a.q_heads + a.k_heads;
      const long long items = static_cast<long long>(a.tokens) * ((heads + kRows - 1) / kRows);
      const long long per = kThreads / kLanes;
      const int blocks = static_cast<int>(std::min<long long>(backward_blocks(), (items + per - 1) / per));
      if (items > 0x7fffffffll - static_cast<long long>(blocks) * per) return cudaErrorInvalidValue;
      if (blocks > 0) {
        norm_rope_backward_kernel<T, W, kLanes, kRows><<<blocks, kThreads, kThreads / kLanes * 2 * a.dim * sizeof(float), s>>>(
            norm_rope_args<T, W>(a), static_cast<const T *>(gq), static_cast<const T *>(gk), static_cast<T *>(dq),
            static_cast<T *>(dk), workspace);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
      }
      norm_rope_weights_kernel<W><<<(2 * a.dim + 31) / 32, 1024, 0, s>>>(workspace, blocks, a.dim, static_cast<W *>(dq_weight),
                                                                     static_cast<W *>(dk_weight));
      return cudaGetLastError();
    });
  });
}

int kv_cache_write(const KvCacheArgs &c, const void *k, const void *v, long long k_token, long long k_head,
                   long long v_token, long long v_head, const void *slots, int wide_slots, int tokens, int type,
                   void *stream) {
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
          const unsigned blocks = blocks_for((static_cast<long long>(tokens) + kRows - 1) / kRows * 2 * c.kv_heads, kLanes);
          if (!blocks) return cudaErrorInvalidValue;
          kv_write_kernel<T, C, kLanes, kRows><<<blocks, kThreads, 0, s>>>(
              cache, static_cast<const T *>(k), static_cast<const T *>(v), k_token, k_head, v_token, v_head, slots,
              wide_slots, tokens);
          return cudaGetLastError();
        };
        return rows <= static_cast<long long>(device_sm_count()) * (2048 / kLanes) ? launch(Int<1>{}) : launch(Int<4>{});
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
          const unsigned blocks = blocks_for((static_cast<long long>(tokens) + kRows - 1) / kRows * 2 * c.kv_heads, kLanes);
          if (!blocks) return cudaErrorInvalidValue;
          kv_read_kernel<T, C, kLanes, kRows><<<blocks, kThreads, 0, s>>>(cache, static_cast<T *>(k_out),
                                                                         static_cast<T *>(v_out), slots, wide_slots, tokens);
          return cudaGetLastError();
        };
        return rows <= static_cast<long long>(device_sm_count()) * (2048 / kLanes) ? launch(Int<1>{}) : launch(Int<4>{});
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
