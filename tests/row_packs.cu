// The places that a thread of a block gets of rows that it shares out (each_pack), on the CPU:
// how many of them, and whether they are the thread's own, in order.  Prints the count.
#include <cstdio>
#include <cstdlib>

#include "dense.cuh"

int main(int, char** argument) {
  const unsigned begin = std::strtoul(argument[1], nullptr, 0), end = std::strtoul(argument[2], nullptr, 0);
  const unsigned rows = std::strtoul(argument[3], nullptr, 0), thread = std::strtoul(argument[4], nullptr, 0);
  const unsigned long long most = std::strtoull(argument[5], nullptr, 0);      // places, and no end beyond them
  unsigned long long places = 0, sum = 0;
  eps_b200::dense::each_pack<8>(begin, end, rows, thread, 256, [&](const unsigned (&row)[8], const unsigned (&pack)[8], const bool (&there)[8]) {
    if (places > most) std::exit(1);
    for (unsigned j = 0; j < 8; ++j) {
      if (row[j] >= rows || pack[j] < begin || pack[j] >= end) std::exit(2);
      if (there[j]) ++places, sum += row[j] * 3ull + pack[j];
    }
  });
  std::printf("%llu %llu\n", places, sum);
  return 0;
}
