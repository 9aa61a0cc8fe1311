// Prints what make_rope makes of the rotations on its standard input, one a line:
// dim base scaling factor original low high gain, then dim / 2 divisors or none.
// Out: "refused", or the gain and the frequencies' 64-bit fractions of a turn.
#include <cstdio>
#include <iostream>
#include <sstream>
#include <string>
#include <vector>

#include "rope_turns.h"

int main() {
  std::string line;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    int dim, scaling, original;
    double base, factor, low, high, gain, f;
    in >> dim >> base >> scaling >> factor >> original >> low >> high >> gain;
    std::vector<float> ff;
    while (in >> f) ff.push_back((float)f);
    kc::RopeParams r;
    if (!kc::make_rope(r, dim, false, (float)base, scaling, (float)factor, original, (float)low, (float)high, (float)gain,
                       ff.empty() ? nullptr : ff.data())) {
      std::puts("refused");
      continue;
    }
    std::printf("%.9g", r.gain);
    for (int i = 0; i < dim / 2; ++i) std::printf(" %llu", (unsigned long long)r.turn[i]);
    std::puts("");
  }
}
