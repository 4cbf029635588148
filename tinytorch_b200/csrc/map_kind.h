// Which lengths of a sequence a tensor map can be given (see packed_plan.cu), found out from the driver's own maps.  Host code without CUDA.
#pragma once
#include <cstdint>
#include <cstring>

namespace ttattn {

// Whether two maps of the same memory differ in nothing but the number of rows (which lies in one of their words).
template <typename Map>
bool same_kind(const Map& a, const Map& b) {
  uint64_t x[sizeof(Map) / 8], y[sizeof(Map) / 8];
  std::memcpy(x, &a, sizeof(x)), std::memcpy(y, &b, sizeof(y));
  int differ = 0;
  for (size_t i = 0; i < sizeof(Map) / 8; ++i) differ += x[i] != y[i];
  return differ <= 1;
}

enum class MapKinds { kFound, kNotEncoded, kNotUnderstood };

// *n: from how many rows on a map is of the kind of `whole`, the map of all `rows`; with fewer it is of the kind of `one`, that of a single row.
// `guess` is tried first; should a driver see it otherwise, n is searched for.  Either way the maps on both sides of the border are compared with the two that
// lengths will be put into: if either is of another kind still (a layout with the rows in two words, say, or with more than one border),
// the driver's maps are not understood, and no length but those two may be put into them.  encode(map, rows): the driver's map of so many rows.
template <typename Map, typename Encode>
MapKinds long_rows(Encode encode, int rows, int64_t guess, const Map& whole, const Map& one, int* n) {
  *n = 1;
  if (same_kind(whole, one)) return MapKinds::kFound;
  Map at, below;
  auto border = [&](int64_t x) { return encode(&at, static_cast<int>(x)) && encode(&below, static_cast<int>(x - 1)); };
  int64_t hi = guess;
  if (hi < 2 || hi > rows || !border(hi) || !same_kind(at, whole) || !same_kind(below, one)) {
    int64_t lo = 1;
    for (hi = rows; hi - lo > 1;) {
      const int64_t mid = (lo + hi) / 2;
      if (!encode(&at, static_cast<int>(mid))) return MapKinds::kNotEncoded;
      (same_kind(at, whole) ? hi : lo) = mid;
    }
    if (!border(hi)) return MapKinds::kNotEncoded;
    if (!same_kind(at, whole) || !same_kind(below, one)) return MapKinds::kNotUnderstood;
  }
  *n = static_cast<int>(hi);
  return MapKinds::kFound;
}

}  // namespace ttattn
