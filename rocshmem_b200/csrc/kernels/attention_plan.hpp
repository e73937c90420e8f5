// Arithmetic of paged attention that the host launcher, the kernels and a CPU test share: how a batch of sequences is
// cut into tiles of keys, how the tiles are dealt to blocks, and where a row of the cache lies.
//
// The tiles of all (sequence, unit) pairs stand in one line: sequence by sequence, within it unit by unit (a unit is a
// key head and up to 8 * NT of its query heads), within that tile by tile. Warp c of the grid takes the share [c * per,
// (c + 1) * per) of the line, whatever pairs its tiles belong to. A pair that lies in one share is finished there; one
// that lies in several leaves a partial result in each of them. A share has at most two such pairs, its first and its
// last, so two places a share hold all partial results whatever the lengths are.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define ATTN_HD __host__ __device__ __forceinline__
#else
#define ATTN_HD inline
#endif

namespace rocshmem {
namespace kernels {
namespace attn {

// The positions [first, end) that a sequence's new token sees. Lengths below zero count as zero, those past the end of
// the block table as its end; window > 0 leaves the last `window` positions.
struct Span {
  int first, end;
};
ATTN_HD Span visible(int length, int capacity, int window) {
  const int end = length < 0 ? 0 : (length > capacity ? capacity : length);
  return Span{window > 0 && end > window ? end - window : 0, end};
}

ATTN_HD int tiles_of(Span s, int tile_keys) { return (s.end - s.first + tile_keys - 1) / tile_keys; }

// Tiles of a share: an equal part of the line, but not fewer than `least` (a share's fixed costs).
ATTN_HD long long per_share(long long total, int shares, int least) {
  const long long per = (total + shares - 1) / shares;
  return per < least ? least : per;
}

// The shares that a pair lies in whose tiles are [begin, begin + n), n > 0.
struct Owners {
  long long first, last;
};
ATTN_HD Owners owners(long long begin, int n, long long per) { return Owners{begin / per, (begin + n - 1) / per}; }

// Which of share c's two places holds its partial result of a pair that begins in share `first`: 0 for a pair that an
// earlier share began, 1 for one that a later share ends.
ATTN_HD int place(long long first, long long c) { return c > first ? 0 : 1; }

// The last share that a pair of n tiles lies in which begins in share `share` with `left` of the share's tiles left.
ATTN_HD int last_share(int share, int n, int left, int per) { return n > left ? share + (n - left + per - 1) / per
    : share; }

// Division of numbers below 2^31 by one divisor, by a multiplication (Granlund and Montgomery): with l = ceil(log2 d)
// and m = floor(2^32 (2^l - d) / d) + 1, n / d = (floor(m n / 2^32) + n) >> l. A division proper takes 20 instructions,
// as many as a fifth of what a row of a cache write needs.
struct Divisor {
  uint32_t d, m, l;
};
inline Divisor divisor(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  return Divisor{d, static_cast<uint32_t>(((1ull << 32) * ((1ull << l) - d)) / d + 1), l};
}
ATTN_HD uint32_t divide(uint32_t n, const Divisor &v) {
  return (static_cast<uint32_t>((static_cast<unsigned long long>(v.m) * n) >> 32) + n) >> v.l;
}

// Row (of `dim` elements) of position `pos` in a cache [pages, kv_heads, page_size, dim], or -1 where the position is
// not visible or its page is no page of the cache. page_size = 1 << shift.
ATTN_HD int page_row(int page, int num_pages, int pos, int shift, int kv_heads, int head) {
  if (page < 0 || page >= num_pages) return -1;
  return ((page * kv_heads + head) << shift) + (pos & ((1 << shift) - 1));
}

// The same for a flat slot (page * page_size + offset), or -1 for a slot outside the cache, which has at most 2^31 - 1
// rows.
ATTN_HD int slot_row(long long slot, int num_slots, int shift, int kv_heads, int head) {
  if (slot < 0 || slot >= num_slots) return -1;
  const int s = static_cast<int>(slot);
  return (((s >> shift) * kv_heads + head) << shift) + (s & ((1 << shift) - 1));
}

}  // namespace attn
}  // namespace kernels
}  // namespace rocshmem
