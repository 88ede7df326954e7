// Which rows of a packed sequence the gradient of its keys goes over.  Row i G + g
// is query i of head g of a group of G; numbers of rows are below 2^31 - 2^14.
#pragma once
#include <hip/hip_runtime.h>

namespace bc2n {

// The first row that sees key j, or the last key for one past it.  (Compared with a row
// this needs no division by the group's heads for each.)
__host__ __device__ constexpr int first_row(bool causal, int j, int lq, int lk, int G) {
  const int i = (j < lk ? j : lk - 1) - (lk - lq);  // below lq
  return causal && i > 0 ? i * G : 0;
}

struct KeyRows {
  int all = 0;    // the sequence's rows
  int first = 0;  // the first that sees a key from j0 on, down to a multiple of the tile
  int blind = 0;  // rows before it see no key at all
};
// Of the keys from j0 on.  Those past the sequence's length have none, wherever in
// a buffer's capacity they lie: j0 times G is bounded by rows only for j0 < lk.
__host__ __device__ constexpr KeyRows rows_of_keys(bool causal, int j0, int lq, int lk, int G, int tile) {
  KeyRows r;
  if (j0 >= lk) return r;
  r.all = lq * G;
  if (!causal) return r;
  const int lag = lk - lq;  // query i sees keys up to i + lag
  r.first = first_row(causal, j0, lq, lk, G) / tile * tile;
  r.blind = (lag < 0 ? -lag : 0) * G;
  return r;
}

struct Part {
  int from = 0, to = 0;
};
// The part-th of `parts` equal ones of them, whole tiles each.
__host__ __device__ constexpr Part part_of_rows(const KeyRows& r, int parts, int part, int tile) {
  const int per = ((r.all - r.first + tile - 1) / tile + parts - 1) / parts * tile;
  Part p;
  p.from = r.first + part * per < r.all ? r.first + part * per : r.all;
  p.to = p.from + per < r.all ? p.from + per : r.all;
  return p;
}

}  // namespace bc2n
