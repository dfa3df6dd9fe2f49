// How the tiles of a batch's query rows are cut along their keys: plain
// arithmetic, used by the plan on the GPU.
#pragma once

namespace bmx {

// Blocks of a piece at most, of tiles with `sum` blocks in all (up to 2^30) and
// `most` in the largest: half as many again as each of the `per_head` workgroups
// of a kv head has to do on average, and at least 4.  A tile is cut only if it is
// longer than that, so the pieces of all cut tiles number less than twice
// per_head: nb / size + 1 < 2 nb / size of each, and size >= 4/3 sum / per_head.
constexpr int piece_size(int sum, int per_head, int most) {
  const int average = (sum + per_head - 1) / per_head, size = average + average / 2;  // (below 2^31)
  const int least = size < 4 ? 4 : size;
  return least < most ? least : most;
}

// Pieces of a tile of nb blocks, of `len` each (the last the rest)
constexpr int piece_count(int nb, int size, int* len) {
  const int n = nb > size ? (nb + size - 1) / size : 1;
  *len = (nb + n - 1) / n;
  return *len > 0 ? (nb + *len - 1) / *len : 1;
}

}  // namespace bmx
