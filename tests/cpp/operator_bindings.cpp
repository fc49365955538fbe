// What an operator launch says about its arguments before anything touches a device: reads a kernel binary and lines
//   <tiling word> ... | <address>:<bytes> ...
// from standard input and prints the launch's answer to each.
#include <cstdint>
#include <cstdio>
#include <fstream>
#include <iostream>
#include <iterator>
#include <sstream>
#include <string>
#include <vector>

#include "runtime/launcher.h"

int main(int argc, char **argv) {
  if (argc != 2) return 2;
  std::ifstream is(argv[1], std::ios::binary);
  const std::vector<uint8_t> binary((std::istreambuf_iterator<char>(is)), std::istreambuf_iterator<char>());
  afir::LaunchDescriptor d;
  if (afir::Status s = afir::parseDescriptorBinary(binary.data(), binary.size(), d); !s) {
    std::printf("descriptor: %s\n", s.message().c_str());
    return 0;
  }
  std::string line;
  while (std::getline(std::cin, line)) {
    std::istringstream words(line);
    std::string w;
    std::vector<int64_t> tiling;
    afir::LaunchArgs args;
    bool behind = false;
    while (words >> w) {
      if (w == "|") behind = true;
      else if (!behind) tiling.push_back(std::stoll(w));
      else {
        const size_t colon = w.find(':');
        args.argPtrs.push_back(reinterpret_cast<void *>(static_cast<uintptr_t>(std::stoull(w.substr(0, colon)))));
        args.argBytes.push_back(std::stoull(w.substr(colon + 1)));
      }
    }
    std::map<std::string, int64_t> values;
    afir::LaunchInfo info;
    afir::Status s = afir::unpackTiling(d, reinterpret_cast<const uint8_t *>(tiling.data()), tiling.size() * 8, values);
    if (s) s = afir::launchDescriptor(d, values, args, info);
    std::printf("%s\n", s ? "launched" : s.message().c_str());
  }
  return 0;
}
