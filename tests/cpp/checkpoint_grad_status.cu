// How a time-out of the checkpoint gradient reaches its caller: the device's words are set by hand, as a wait that runs out
// would set them, and the executor's answers are compared with what they have to be.
//   <program> <checkpoint gradient: binary, tiling> <matmul: binary, tiling>
#include "kernels/checkpoint_grad_tcgen05.cu"

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <fstream>
#include <iterator>
#include <string>
#include <vector>

#include "runtime/executor.h"

namespace {

constexpr int T = 64, D = 128, N = 256;  // and a matmul of 256 x 256 x 256

std::vector<uint8_t> fileOf(const char *path) {
  std::ifstream is(path, std::ios::binary);
  return std::vector<uint8_t>((std::istreambuf_iterator<char>(is)), std::istreambuf_iterator<char>());
}
void must(cudaError_t e) {
  if (e == cudaSuccess) return;
  std::printf("CUDA: %s\n", cudaGetErrorString(e));
  std::exit(3);
}
int failures = 0;
void expect(const char *what, const afir::Status &s, const char *words) {
  const bool good = words ? !s && s.message().find(words) != std::string::npos : s.ok();
  if (!good) {
    ++failures;
    std::printf("%s: %s\n", what, s ? "no error" : s.message().c_str());
  }
}
void setWord(int word, unsigned int value) {
  must(cudaDeviceSynchronize());
  must(cudaMemcpyToSymbol(afir::kernels::checkpointGradStatusWords, &value, sizeof(value), static_cast<size_t>(word) * sizeof(value)));
}

struct Kernel {
  std::vector<uint8_t> binary, tiling;
  std::string name;
  std::vector<const void *> in;
  std::vector<size_t> inBytes;
  std::vector<void *> out;
  std::vector<size_t> outBytes;
  void *workspace = nullptr;

  void input(size_t bytes) {
    void *p;
    must(cudaMalloc(&p, bytes));
    must(cudaMemset(p, 0, bytes));
    in.push_back(p);
    inBytes.push_back(bytes);
  }
  void output(size_t bytes) {
    void *p;
    must(cudaMalloc(&p, bytes));
    out.push_back(p);
    outBytes.push_back(bytes);
  }
  afir::Status launch(afir::CudaExecutor &e, cudaStream_t stream) {
    afir::RunRequest r;
    r.binary = binary.data();
    r.binaryLen = binary.size();
    r.functionName = name;
    r.numInputs = static_cast<int>(in.size());
    r.inputPtrs = in.data();
    r.inputBytes = inBytes.data();
    r.numOutputs = static_cast<int>(out.size());
    r.outputPtrs = out.data();
    r.outputBytes = outBytes.data();
    r.tiling = tiling.data();
    r.tilingLen = tiling.size();
    return e.launchDevice(r, workspace, workspace ? 4096 : 0, stream);
  }
};

} // namespace

int main(int argc, char **argv) {
  if (argc != 5) return 2;
  Kernel gradient, product;
  gradient.binary = fileOf(argv[1]);
  gradient.tiling = fileOf(argv[2]);
  gradient.name = "checkpoint_weight_grad";
  gradient.input(T * D);
  gradient.input(T);
  gradient.input(T * N * 2);
  gradient.output(D * N * 2);
  must(cudaMalloc(&gradient.workspace, 4096));
  product.binary = fileOf(argv[3]);
  product.tiling = fileOf(argv[4]);
  product.name = "product";
  product.input(256 * 256 * 2);
  product.input(256 * 256 * 2);
  product.input(256 * 2);
  product.output(256 * 256 * 2);
  must(cudaMalloc(&product.workspace, 4096));
  must(cudaDeviceSynchronize());
  cudaStream_t stream;
  must(cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking));

  afir::CudaExecutor first, second;
  expect("initialize", first.initialize(0), nullptr);
  expect("initialize", second.initialize(0), nullptr);

  // a launch of another kernel behind it, with its own workspace, does not hide a time-out; it is reported once
  expect("gradient", gradient.launch(first, stream), nullptr);
  setWord(0, 0x103);
  expect("matmul", product.launch(first, stream), nullptr);
  expect("behind a matmul", first.synchronize(stream), "checkpoint gradient: conversion gave up");
  expect("told once", first.synchronize(stream), nullptr);

  // what the workspace holds is no report, fresh or used before
  for (int i = 0; i < 2; ++i) {
    must(cudaMemset(gradient.workspace, 0xff, 4096));
    must(cudaDeviceSynchronize());
    expect("gradient", gradient.launch(first, stream), nullptr);
  }
  expect("a workspace's old bytes", first.synchronize(stream), nullptr);

  // executors do not read each other's
  expect("gradient", gradient.launch(first, stream), nullptr);
  expect("gradient", gradient.launch(second, stream), nullptr);
  setWord(0, 0x100);
  expect("the other executor", second.synchronize(stream), nullptr);
  expect("this executor", first.synchronize(stream), "checkpoint gradient: TMA producer gave up");

  // a replayed graph: no workspace, captured before anything ran on this executor; every replay is looked at
  afir::CudaExecutor third;
  expect("initialize", third.initialize(0), nullptr);
  gradient.workspace = nullptr;
  cudaGraph_t graph;
  cudaGraphExec_t exec;
  must(cudaStreamBeginCapture(stream, cudaStreamCaptureModeGlobal));
  expect("captured", gradient.launch(third, stream), nullptr);
  must(cudaStreamEndCapture(stream, &graph));
  must(cudaGraphInstantiate(&exec, graph, 0));
  for (int i = 0; i < 2; ++i) {
    must(cudaGraphLaunch(exec, stream));
    expect("replayed", third.synchronize(stream), nullptr);
    setWord(2, 0x101);
    must(cudaGraphLaunch(exec, stream));
    expect("replayed and timed out", third.synchronize(stream), "checkpoint gradient: MMA issuer gave up");
  }
  must(cudaDeviceSynchronize());
  std::printf("%d failures\n", failures);
  return failures ? 1 : 0;
}
