// What an operator launch says about its workspace before anything touches a device: reads a kernel binary and lines
//   <tiling word> ... | <address>:<bytes> ... | <workspace address>:<bytes>
// from standard input and prints the launch's answer to each.
#include <cstdint>
#include <cstdio>
#include <fstream>
#include <iostream>
#include <iterator>
#include <sstream>
#include <string>
#include <tuple>
#include <utility>
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
  auto range = [](const std::string &w) {
    const size_t colon = w.find(':');
    return std::make_pair(reinterpret_cast<void *>(static_cast<uintptr_t>(std::stoull(w.substr(0, colon)))), static_cast<size_t>(std::stoull(w.substr(colon + 1))));
  };
  std::string line, w;
  while (std::getline(std::cin, line)) {
    std::istringstream words(line);
    std::vector<int64_t> tiling;
    afir::LaunchArgs args;
    int part = 0;
    while (words >> w) {
      if (w == "|") ++part;
      else if (part == 0) tiling.push_back(std::stoll(w));
      else if (part == 1) {
        args.argPtrs.push_back(range(w).first);
        args.argBytes.push_back(range(w).second);
      } else std::tie(args.workspace, args.workspaceBytes) = range(w);
    }
    std::map<std::string, int64_t> values;
    afir::LaunchInfo info;
    afir::Status s = afir::unpackTiling(d, reinterpret_cast<const uint8_t *>(tiling.data()), tiling.size() * 8, values);
    size_t need = 0;
    if (s) s = afir::requiredWorkspaceBytes(d, values, 0, need);
    if (s) s = afir::launchDescriptor(d, values, args, info);
    std::printf("%zu %s\n", need, s ? "launched" : s.message().c_str());
  }
  return 0;
}
