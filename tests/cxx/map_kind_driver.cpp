// Border of short and long tensor maps (csrc/map_kind.h) against encoders of several layouts; prints what each case gives.
#include <cstdio>
#include <cstdlib>

#include "../../tinytorch_b200/csrc/map_kind.h"

struct Map {
  uint64_t w[16];
};

int main(int argc, char** argv) {
  if (argc != 5) return 2;
  const int layout = std::atoi(argv[1]), rows = std::atoi(argv[2]), border = std::atoi(argv[3]);
  const long guess = std::atol(argv[4]);
  int calls = 0;
  auto encode = [&](Map* m, int n) {
    ++calls;
    if (n < 1 || n > rows) std::exit(3);  // (beyond the tensor: such a map is not asked for)
    if (layout == 5 && n != rows && n != 1) return false;
    *m = Map{};
    m->w[0] = 0x1234, m->w[4] = static_cast<uint64_t>(n) << 32;
    if (layout == 0 || layout == 2) m->w[1] = n >= border ? 0x200 : 0;              // a bit for long tensors
    if (layout == 2) m->w[2] = n >= 2 * border ? 1 : 0;                             // ... and another for longer ones
    if (layout == 3) m->w[7] = n;                                                   // rows in two words
    if (layout == 4) m->w[1] = n >= border ? 0x200 : 0, m->w[2] = n >= border ? 7 : 0;  // a border that shows in two words
    return true;
  };
  Map whole, one;
  if (!encode(&whole, rows) || !encode(&one, 1)) return 4;
  if (layout == 5) whole.w[1] = 0x200;  // (the driver refuses what lies between)
  calls = 0;
  int n = -1;
  const auto found = ttattn::long_rows<Map>(encode, rows, guess, whole, one, &n);
  std::printf("%d %d %d\n", static_cast<int>(found), n, calls);
  return 0;
}
