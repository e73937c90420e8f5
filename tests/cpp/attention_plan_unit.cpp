// The arithmetic of paged attention's split (attention_plan.hpp) on the CPU: every tile of every pair is taken by
// exactly one share, in order; partial results of one pair lie in places of their own; rows of pages that do not exist
// are refused.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <utility>
#include <vector>

#include "kernels/attention_plan.hpp"

using namespace rocshmem::kernels::attn;

#define CHECK(cond)                                                     \
  do {                                                                  \
    if (!(cond)) {                                                      \
      std::fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #cond);   \
      std::exit(1);                                                     \
    }                                                                   \
  } while (0)

namespace {

void check_spans() {
  CHECK(visible(-3, 100, 0).end == 0);
  CHECK(visible(-3, 100, 0).first == 0);
  CHECK(visible(500, 100, 0).end == 100);
  CHECK(visible(50, 100, 20).first == 30 && visible(50, 100, 20).end == 50);
  CHECK(visible(20, 100, 20).first == 0);
  CHECK(visible(5, 100, 20).first == 0);
  CHECK(tiles_of(visible(0, 100, 0), 64) == 0);
  CHECK(tiles_of(visible(1, 100, 0), 64) == 1);
  CHECK(tiles_of(visible(64, 100, 0), 64) == 1);
  CHECK(tiles_of(visible(65, 100, 0), 64) == 2);
  CHECK(tiles_of(visible(0x7fffff00, 0x7fffff00, 0), 128) == 0x7fffff00 / 128);
}

void check_rows() {
  CHECK(page_row(-1, 8, 5, 4, 2, 1) == -1);
  CHECK(page_row(8, 8, 5, 4, 2, 1) == -1);
  CHECK(page_row(-2147483647 - 1, 8, 5, 4, 2, 1) == -1);
  CHECK(page_row(2147483647, 8, 5, 4, 2, 1) == -1);
  CHECK(page_row(7, 8, 16 + 5, 4, 2, 1) == ((7 * 2 + 1) << 4) + 5);
  CHECK(page_row(3, 4, 9, 0, 1, 0) == 3);
  CHECK(slot_row(-1, 64, 4, 2, 1) == -1);
  CHECK(slot_row(64, 64, 4, 2, 1) == -1);
  CHECK(slot_row(1ll << 40, 64, 4, 2, 1) == -1);
  CHECK(slot_row(63, 64, 4, 2, 1) == ((3 * 2 + 1) << 4) + 15);
  CHECK(slot_row((1ll << 32) + 5, 64, 4, 2, 1) == -1);  // not what its low 32 bits say
  // The last row of the largest cache, 2^31 - 32 rows in pages of 16 slots and two heads.
  const int slots = 0x7fffffe0 / 2;
  CHECK(slot_row(slots - 1, slots, 4, 2, 1) == 0x7fffffe0 - 1);
  CHECK(slot_row(slots, slots, 4, 2, 1) == -1);
}

void check_division() {
  std::mt19937 rng(9);
  for (uint32_t d = 1; d < 5000; ++d) {
    const Divisor v = divisor(d);
    for (uint32_t n : {0u, 1u, d - 1, d, d + 1, 2 * d - 1, 2 * d, 0x7fffffffu, 0x7fffffffu - d, 0x7fffffffu / d * d,
        0x7fffffffu / d * d - 1,
                       static_cast<uint32_t>(rng() >> 1), static_cast<uint32_t>(rng() >> 9), static_cast<uint32_t>(rng() >> 20)}) {
      if (n <= 0x7fffffffu) CHECK(divide(n, v) == n / d);
    }
  }
  for (uint32_t d : {1u << 20, (1u << 20) + 1, (1u << 21) - 1, 1u << 21, 0x7ffffffeu, 0x7fffffffu}) {
    for (uint32_t n : {0u, d - 1, d, 0x7fffffffu}) CHECK(divide(n, divisor(d)) == n / d);
  }
}

void check_split(const std::vector<int> &lengths, int capacity, int window, int units, int shares, int least,
    int tile) {
  std::vector<long long> bases;
  long long total = 0;
  for (int n : lengths) {
    bases.push_back(total);
    total += static_cast<long long>(tiles_of(visible(n, capacity, window), tile)) * units;
  }
  const long long per = per_share(total, shares, least);
  CHECK(per >= least && per * shares >= total);
  std::set<std::pair<long long, int>> places;
  for (size_t b = 0; b < lengths.size(); ++b) {
    const int n = tiles_of(visible(lengths[b], capacity, window), tile);
    for (int u = 0; u < units && n > 0; ++u) {
      const long long begin = bases[b] + static_cast<long long>(u) * n;
      const Owners own = owners(begin, n, per);
      CHECK(own.first >= 0 && own.first <= own.last && own.last < shares);
      const long long left = ((own.first + 1) * per < total ? (own.first + 1) * per : total) - begin;
      CHECK(last_share(static_cast<int>(own.first), n, static_cast<int>(left), static_cast<int>(per)) == own.last);
      // The tiles that the owners' shares hold of this pair are all of them.
      long long seen = 0;
      for (long long c = own.first; c <= own.last; ++c) {
        const long long lo = c * per > begin ? c * per : begin;
        const long long hi = (c + 1) * per < begin + n ? (c + 1) * per : begin + n;
        CHECK(hi > lo);
        seen += hi - lo;
        if (own.first == own.last) continue;
        // What the warp itself goes by: it begins the pair (place 1) or finds it begun (place 0).
        CHECK(place(own.first, c) == (lo == begin ? 1 : 0));
        CHECK(places.insert({c, place(own.first, c)}).second);
      }
      CHECK(seen == n);
    }
  }
}

}  // namespace

int main() {
  check_spans();
  check_rows();
  check_division();
  std::mt19937 rng(5);
  for (int round = 0; round < 3000; ++round) {
    std::vector<int> lengths(1 + rng() % 40);
    const int most = 1 << (rng() % 14);
    for (int &n : lengths) n = rng() % 5 == 0 ? 0 : static_cast<int>(rng() % (most + 2)) - 1;
    const int window = rng() % 3 == 0 ? 1 + rng() % most : 0;
    check_split(lengths, most, window, 1 + rng() % 9, 1 + rng() % 300, 1 + rng() % 6, rng() % 2 ? 16 : 32);
  }
  check_split({1000000, 0, 1}, 1 << 20, 0, 1, 1184, 4, 16);
  check_split({0, 0}, 64, 0, 3, 1184, 4, 16);
  std::puts("ok");
  return 0;
}
