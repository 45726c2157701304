// Host-only: how many parts the orthogonalised updates take, by steps and coefficients.
#include <cstdio>
#include <cstdlib>

#include "ortho_update.hip"

int main(int argc, char **argv) {  // type, weights, then steps a b c, any number of times
  const cavs_ortho_desc d{4, 4, argv, 4, nullptr, 0, std::atoi(argv[2]) ? reinterpret_cast<float *>(argv) : nullptr, 4, argv, 4};
  for (int i = 3; i + 3 < argc; i += 4) {
    cavs_ortho_options o{std::atoi(argv[i]), 1, std::strtof(argv[i + 1], nullptr), std::strtof(argv[i + 2], nullptr), std::strtof(argv[i + 3], nullptr)};
    std::printf("%d\n", two_parts(std::atoi(argv[1]), 1, &d, o) ? 2 : 3);
  }
  return 0;
}
